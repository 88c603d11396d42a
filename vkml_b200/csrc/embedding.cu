// Embedding lookup with scaling, and its gradient.
//
//   rows[t] = scale * table[ids[t]]                                    t = 0 .. N-1
//   table[v] = scale * sum over t with ids[t] = v of rows[t]           v = 0 .. V-1 (backward)
//
// Both are bound by memory: the lookup by N rows written and as many read, the gradient by N rows read and V rows
// written.  Table and rows are F32 or F16 each; sums are held in F32 and rounded once.
#include "operators.cuh"

#include <algorithm>

namespace b200 {
namespace {

constexpr int kThreads = 256;

// The token ids: [outer, inner] with any strides.
struct Ids {
    RowsArg at;
    FastDiv inner;
    int wide;  // I64

    __device__ __forceinline__ int64_t operator[](uint32_t t) const { return load_index(row_at(at, inner, t), wide != 0); }
};

// ---- lookup -----------------------------------------------------------------

// A thread moves kItems pieces of a row, kThreads pieces apart, so that their ids and then their elements are all under way together.
// A piece is 8 elements where rows of both sides start on 16 bytes and hold whole pieces, one element otherwise.
constexpr int kItems = 4;

template <typename TI, typename TO, bool WIDE>
__global__ void __launch_bounds__(kThreads)
lookup_kernel(RowsArg out, const char* table, int64_t pitch, Ids ids, int64_t vocab, FastDiv pieces, int64_t total, float scale, uint32_t* status) {
    pdl_prologue();
    const int64_t first = int64_t(blockIdx.x) * (kThreads * kItems) + threadIdx.x;
    uint32_t token[kItems], piece[kItems];
    int64_t id[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int64_t i = first + k * kThreads;
        id[k] = -2;
        if (i < total) {
            if (total < (int64_t(1) << 31)) {
                pieces.divmod(static_cast<uint32_t>(i), token[k], piece[k]);
            } else {
                token[k] = static_cast<uint32_t>(i / pieces.d);
                piece[k] = static_cast<uint32_t>(i - int64_t(token[k]) * pieces.d);
            }
            id[k] = ids[token[k]];
            if (id[k] < 0 || id[k] >= vocab) {
                id[k] = -1;
                if (piece[k] == 0) atomicOr(status, kStatusIndexOutOfRange);
            }
        }
    }
    if constexpr (WIDE) {
        Raw8<TI> raw[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (id[k] >= 0) load8(raw[k], reinterpret_cast<const TI*>(table + id[k] * pitch) + int64_t(piece[k]) * 8);
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (id[k] == -2) continue;
            float x[8] = {};
            if (id[k] >= 0) {
                unpack8(raw[k], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= scale;
            }
            store8(reinterpret_cast<TO*>(row_at(out, ids.inner, token[k])) + int64_t(piece[k]) * 8, x);
        }
    } else {
        TI raw[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (id[k] >= 0) raw[k] = reinterpret_cast<const TI*>(table + id[k] * pitch)[piece[k]];
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (id[k] == -2) continue;
            reinterpret_cast<TO*>(row_at(out, ids.inner, token[k]))[piece[k]] = from_float<TO>(id[k] >= 0 ? to_float(raw[k]) * scale : 0.f);
        }
    }
}

// ---- gradient: rows of the table owned by blocks ------------------------------

// A block owns `owned` rows of the table and up to kThreads * 4 columns of them, as sums in shared memory.  It reads all ids, a chunk at a
// time and in order, lists the tokens of its rows, and adds their rows to the sums: each column has one thread and each list ascends, so
// the order of addition is the tokens' and the result does not depend on which block does what.  One launch, no scratch.
constexpr int kChunk = 1024;

template <typename TG, typename TO>
__global__ void __launch_bounds__(kThreads)
owned_rows_kernel(char* table, int64_t pitch, RowsArg grad, Ids ids, uint32_t count, int64_t vocab, int64_t width, int owned, int columns,
                  int64_t padding, float scale, int accumulate, uint32_t* status) {
    extern __shared__ float sums[];  // [owned][columns]
    __shared__ uint32_t list_token[kChunk];
    __shared__ uint16_t list_row[kChunk];
    __shared__ uint32_t touched[32];  // of `owned` <= 1024 rows
    __shared__ int warp_count[kChunk / 32];
    pdl_prologue();
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int64_t row0 = int64_t(blockIdx.x) * owned;
    const int rows = static_cast<int>(min(int64_t(owned), vocab - row0));
    const int64_t col0 = int64_t(blockIdx.y) * columns;
    const int cols = static_cast<int>(min(int64_t(columns), width - col0));
    for (int i = tid; i < rows * columns; i += kThreads) sums[i] = 0.f;
    if (tid < 32) touched[tid] = 0;
    for (uint32_t base = 0; base < count; base += kChunk) {
        __syncthreads();
        uint32_t mine[kChunk / kThreads];
        int64_t row[kChunk / kThreads];
#pragma unroll
        for (int k = 0; k < kChunk / kThreads; ++k) {
            const uint32_t t = base + k * kThreads + tid;
            row[k] = -1;
            if (t < count) {
                const int64_t id = ids[t];
                if (id >= row0 && id < row0 + rows && id != padding) {
                    row[k] = id - row0;
                } else if ((id < 0 || id >= vocab) && id != padding && blockIdx.x == 0 && blockIdx.y == 0) {
                    atomicOr(status, kStatusIndexOutOfRange);
                }
            }
            mine[k] = __ballot_sync(0xffffffffu, row[k] >= 0);
            if (lane == 0) warp_count[k * (kThreads / 32) + warp] = __popc(mine[k]);
        }
        __syncthreads();
        if (warp == 0) {  // where each warp's tokens go
            int n = lane < kChunk / 32 ? warp_count[lane] : 0, upto = n;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int other = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += other;
            }
            if (lane < kChunk / 32) warp_count[lane] = upto;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kChunk / kThreads; ++k) {
            if (row[k] < 0) continue;
            const int w = k * (kThreads / 32) + warp;
            const int at = (w > 0 ? warp_count[w - 1] : 0) + __popc(mine[k] & ((1u << lane) - 1));
            list_token[at] = base + k * kThreads + tid;
            list_row[at] = static_cast<uint16_t>(row[k]);
            atomicOr(&touched[row[k] / 32], 1u << (row[k] % 32));
        }
        __syncthreads();
        const int n = warp_count[kChunk / 32 - 1];
        for (int c = tid; c < cols; c += kThreads) {
            int j = 0;
            for (; j + 4 <= n; j += 4) {  // four rows under way
                float g[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) g[k] = to_float(reinterpret_cast<const TG*>(row_at(grad, ids.inner, list_token[j + k]))[col0 + c]);
#pragma unroll
                for (int k = 0; k < 4; ++k) sums[int(list_row[j + k]) * columns + c] += g[k];
            }
            for (; j < n; ++j) sums[int(list_row[j]) * columns + c] += to_float(reinterpret_cast<const TG*>(row_at(grad, ids.inner, list_token[j]))[col0 + c]);
        }
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
        const bool any = (touched[r / 32] >> (r % 32)) & 1;
        if (accumulate && !any) continue;
        TO* to = reinterpret_cast<TO*>(table + (row0 + r) * pitch) + col0;
        for (int c = tid; c < cols; c += kThreads) {
            float x = sums[r * columns + c] * scale;
            if (accumulate) x += to_float(to[c]);
            to[c] = from_float<TO>(x);
        }
    }
}

struct Problem {
    int64_t count, vocab, width, pitch;
    Ids ids;
    RowsArg rows;
};

// What both directions ask of their arguments.
Problem check_embedding(const b200_embedding_args& a, bool backward) {
    check_rows(a.table, "table");
    if (a.table.ndim != 2) fail(B200_SHAPE_ERROR, "table: rank " + std::to_string(a.table.ndim) + ", 2 is needed");
    check_tensor(a.ids, "ids");
    check_rows(a.rows, "rows");
    if (!is_float(a.table.dtype) || !is_float(a.rows.dtype)) fail(B200_DTYPE_ERROR, "table and rows are F32 or F16");
    if (!is_index(a.ids.dtype)) fail(B200_DTYPE_ERROR, "ids are I64 or I32");
    if (a.ids.ndim > 2) fail(B200_SHAPE_ERROR, "ids: rank " + std::to_string(a.ids.ndim) + " is above 2");
    if (a.rows.ndim != a.ids.ndim + 1 || !same_extents(a.rows, a.ids, a.ids.ndim)) fail(B200_SHAPE_ERROR, "rows have the extents of ids and the table's width");
    Problem p;
    p.vocab = a.table.dims[0];
    p.width = a.table.dims[1];
    if (a.rows.dims[a.rows.ndim - 1] != p.width) fail(B200_SHAPE_ERROR, "rows have the extents of ids and the table's width");
    if (p.vocab >= (int64_t(1) << 31) || p.width >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "table: an extent of 2^31 or more");
    p.pitch = p.vocab > 1 ? a.table.strides[0] : 0;
    const RowShape s = row_shape(a.ids, a.ids.ndim);
    p.count = s.rows;
    if (p.count != 0 && p.vocab == 0) fail(B200_INDEX_ERROR, "embedding: an id into an empty table");
    if (p.count != 0 && a.ids.data == nullptr) fail(B200_INVALID_ARGUMENT, "ids have no storage");
    p.ids.at = rows_arg(a.ids, a.ids.ndim);
    p.ids.inner = FastDiv(static_cast<uint32_t>(std::max<int64_t>(s.inner, 1)));
    p.ids.wide = a.ids.dtype == B200_I64;
    p.rows = rows_arg(a.rows, a.ids.ndim);
    if ((a.flags & ~B200_ACCUMULATE) != 0 || (!backward && a.flags != 0)) fail(B200_INVALID_ARGUMENT, "unknown flags");
    const b200_tensor none{}, scratch = backward ? workspace_tensor(a.workspace, a.workspace_bytes) : none;
    if (backward) check_results({{&a.table, "table"}, {&scratch, "workspace"}}, {{&a.ids, "ids"}, {&a.rows, "rows"}}, {});
    else check_results({{&a.rows, "rows"}}, {{&a.ids, "ids"}, {&a.table, "table"}}, {});
    return p;
}

template <typename Fn>
void with_types(int table, int rows, Fn&& fn) {
    if (table == B200_F32 && rows == B200_F32) fn(float{}, float{});
    else if (table == B200_F32) fn(float{}, __half{});
    else if (rows == B200_F32) fn(__half{}, float{});
    else fn(__half{}, __half{});
}

void launch_lookup(b200_ctx* ctx, const b200_embedding_args& a) {
    const Problem p = check_embedding(a, false);
    if (p.count == 0 || p.width == 0) return;
    wait_for_tensors(ctx, {&a.table, &a.ids, &a.rows});
    const bool wide = p.width % 8 == 0 && aligned_rows(p.rows, 16) && reinterpret_cast<uintptr_t>(a.table.data) % 16 == 0 && p.pitch % 16 == 0;
    const int64_t pieces = wide ? p.width / 8 : p.width, total = p.count * pieces;
    const int64_t blocks = ceil_div(total, kThreads * kItems);
    if (blocks >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "embedding: too many elements");
    ProfScope scope(ctx, "embedding");
    with_types(a.table.dtype, a.rows.dtype, [&](auto ti, auto to) {
        using TI = decltype(ti);
        using TO = decltype(to);
        launch_kernel(ctx, wide ? lookup_kernel<TI, TO, true> : lookup_kernel<TI, TO, false>, static_cast<unsigned>(blocks), kThreads, 0, p.rows,
                      static_cast<const char*>(a.table.data), p.pitch, p.ids, p.vocab, FastDiv(static_cast<uint32_t>(pieces)), total, a.scale, ctx->d_status);
    });
    check_last_launch("embedding");
    ctx->count_launch();
}

void launch_gradient(b200_ctx* ctx, const b200_embedding_args& a) {
    const Problem p = check_embedding(a, true);
    if (p.vocab == 0 || p.width == 0) return;
    wait_for_tensors(ctx, {&a.table, &a.ids, &a.rows});
    ProfScope scope(ctx, "embedding_backward");
    const int columns = static_cast<int>(std::min<int64_t>(p.width, kThreads * 4));
    const int64_t tiles = ceil_div(p.width, columns);
    // rows of sums: 40 KB at most (four blocks to an SM), and few enough that two blocks for each SM have some
    const int64_t most = std::min<int64_t>(1024, std::max<int64_t>(1, 10240 / columns));
    const int owned = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, ceil_div(p.vocab * tiles, sm_count() * 2))));
    const dim3 grid(static_cast<unsigned>(ceil_div(p.vocab, owned)), static_cast<unsigned>(tiles));
    if (tiles > 65535) fail(B200_SHAPE_ERROR, "embedding_backward: a row of more than 65535 * 1024 elements");
    with_types(a.table.dtype, a.rows.dtype, [&](auto to, auto tg) {
        using TO = decltype(to);
        using TG = decltype(tg);
        launch_kernel(ctx, owned_rows_kernel<TG, TO>, grid, kThreads, sizeof(float) * owned * columns, static_cast<char*>(a.table.data), p.pitch, p.rows, p.ids,
                      static_cast<uint32_t>(p.count), p.vocab, p.width, owned, columns, a.padding_id < 0 ? INT64_MIN : a.padding_id, a.scale,
                      static_cast<int>(a.flags & B200_ACCUMULATE), ctx->d_status);
    });
    check_last_launch("embedding_backward");
    ctx->count_launch();
}

}  // namespace

void check_embedding_call(const b200_embedding_args& a, bool backward) { (void)check_embedding(a, backward); }

}  // namespace b200

using namespace b200;

extern "C" {

int b200_embedding(b200_ctx* ctx, const b200_embedding_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_lookup(ctx, *args); });
}

int b200_embedding_backward(b200_ctx* ctx, const b200_embedding_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_gradient(ctx, *args); });
}

int b200_embedding_backward_workspace(const b200_embedding_args* args, size_t* nbytes) {
    if (args == nullptr || nbytes == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(nullptr, [&] {
        (void)check_embedding(*args, true);
        *nbytes = 0;
    });
}

}  // extern "C"
