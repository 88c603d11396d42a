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

// ---- gradient: sorted tokens --------------------------------------------------

// The tokens are sorted by id, those of one id in their own order, by one cluster of blocks: radix passes over 8 bits of the id, each of which counts
// the digits of every warp's stretch of the tokens, adds the counts up over warps (shared memory) and blocks (the cluster's shared memory), and
// moves each token to its place.  Tokens that have no gradient sort behind all others, as id V.  The blocks outside of the first cluster write zeros
// over the table meanwhile: sorting leaves the memory idle.  16 blocks of 1024 threads sort 131072 tokens in the time that writing 130 MB takes.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;

struct SortArgs {
    Ids ids;
    uint2* buffer[2];  // (id, token)
    uint32_t count;
    uint32_t vocab;
    int64_t padding;
    int passes, digit_bits;
    char* table;       // to be filled with zeros: null where not
    int64_t pitch, row_bytes;
    uint32_t* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// A word of shared memory of block `rank` of the cluster, at the address that `mine` has here.
__device__ __forceinline__ uint32_t cluster_load(const uint32_t* mine, uint32_t rank) {
    uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), there, x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(there) : "memory");
    return x;
}

__device__ void fill_zeros(const SortArgs& k, uint32_t block, uint32_t blocks) {
    const uint32_t warp = block * kSortWarps + threadIdx.x / 32, warps = blocks * kSortWarps, lane = threadIdx.x % 32;
    const bool wide = ((reinterpret_cast<uintptr_t>(k.table) | k.pitch | k.row_bytes) & 15) == 0;
    if (wide) {
        // dense rows are one stretch, cut into pieces of 4 KB; others are taken one by one
        const bool dense = k.pitch == k.row_bytes;
        const int64_t piece = dense ? 256 : k.row_bytes / 16, all = dense ? int64_t(k.vocab) * k.row_bytes / 16 : 0;
        const int64_t pieces = dense ? (all + piece - 1) / piece : k.vocab;
        for (int64_t p = warp; p < pieces; p += warps) {
            uint4* to = reinterpret_cast<uint4*>(k.table + (dense ? p * piece * 16 : p * k.pitch));
            const int64_t n = dense ? min(piece, all - p * piece) : piece;
            for (int64_t i = lane; i < n; i += 32) to[i] = make_uint4(0, 0, 0, 0);
        }
    } else {
        for (int64_t r = warp; r < k.vocab; r += warps) {
            uint16_t* to = reinterpret_cast<uint16_t*>(k.table + r * k.pitch);
            for (int64_t i = lane; i < k.row_bytes / 2; i += 32) to[i] = 0;
        }
    }
}

__global__ void __launch_bounds__(kSortThreads) sort_tokens_kernel(const SortArgs k) {
    __shared__ uint32_t place[kSortWarps][256];  // counts of each warp's digits; then where its next token of a digit goes
    __shared__ uint32_t total[256];              // this block's counts, read by the others
    __shared__ uint32_t upto[8];
    pdl_prologue();
    const uint32_t blocks = cluster_blocks(), rank = cluster_rank();
    if (blockIdx.x >= blocks) {
        if (k.table != nullptr) fill_zeros(k, blockIdx.x - blocks, gridDim.x - blocks);
        return;  // (whole clusters)
    }
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    // each warp's stretch: whole groups of 32 tokens
    const uint32_t groups = (k.count + 31) / 32, warps = blocks * kSortWarps, per = (groups + warps - 1) / warps;
    const uint32_t first = min(groups, (rank * kSortWarps + warp) * per), last = min(groups, first + per);
    for (int pass = 0; pass < k.passes; ++pass) {
        const uint2* from = k.buffer[(pass + 1) & 1];
        uint2* to = k.buffer[pass & 1];
        const int shift = pass * k.digit_bits;
        const uint32_t mask = (1u << k.digit_bits) - 1;
        auto token = [&](uint32_t i, bool report) {
            if (pass > 0) return __ldcg(&from[i]);
            const int64_t id = k.ids[i];
            const bool in = id >= 0 && id < int64_t(k.vocab);
            if (report && !in && id != k.padding) atomicOr(k.status, kStatusIndexOutOfRange);
            return make_uint2(in && id != k.padding ? static_cast<uint32_t>(id) : k.vocab, i);
        };
        for (int i = tid; i < kSortWarps * 256; i += kSortThreads) (&place[0][0])[i] = 0;
        __syncthreads();
        for (uint32_t g = first; g < last; ++g) {
            const uint32_t i = g * 32 + lane;
            const uint32_t d = i < k.count ? (token(i, true).x >> shift) & mask : 256u;
            const uint32_t peers = __match_any_sync(0xffffffffu, d);
            if (d < 256 && lane == __ffs(peers) - 1) place[warp][d] += __popc(peers);
            __syncwarp();
        }
        __syncthreads();
        if (tid < 256) {  // exclusive over the warps
            uint32_t sum = 0;
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t n = place[w][tid];
                place[w][tid] = sum;
                sum += n;
            }
            total[tid] = sum;
        }
        cluster_sync();
        if (tid < 256) {  // over the blocks, and over the digits below
            uint32_t all = 0, before = 0;
            for (uint32_t b = 0; b < blocks; ++b) {
                const uint32_t n = cluster_load(&total[tid], b);
                if (b < rank) before += n;
                all += n;
            }
            uint32_t scan = all;
#pragma unroll
            for (int s = 1; s < 32; s *= 2) {
                const uint32_t other = __shfl_up_sync(0xffffffffu, scan, s);
                if (lane >= s) scan += other;
            }
            if (lane == 31) upto[warp] = scan;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int w = 0; w < warp; ++w) scan += upto[w];
            const uint32_t base = scan - all + before;
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) place[w][tid] += base;
        }
        __syncthreads();
        for (uint32_t g = first; g < last; ++g) {
            const uint32_t i = g * 32 + lane;
            const uint2 x = i < k.count ? token(i, false) : make_uint2(0, 0);
            const uint32_t d = i < k.count ? (x.x >> shift) & mask : 256u;
            const uint32_t peers = __match_any_sync(0xffffffffu, d);
            if (d < 256) to[place[warp][d] + __popc(peers & ((1u << lane) - 1))] = x;
            __syncwarp();
            if (d < 256 && lane == __ffs(peers) - 1) place[warp][d] += __popc(peers);
            __syncwarp();
        }
        cluster_sync();  // the moved tokens are there, and no block reads another's counts any more
    }
}

// The sorted tokens are cut into chunks of equal length.  Threads that share a row walk a chunk with a sum for each of their columns; where the id
// changes, the sum is that row of the table, unless the id's tokens reach over an end of the chunk: such a sum is left in `partial`, [chunk][0]
// where they began in an earlier chunk, [chunk][1] where they begin here, and join_kernel adds them up in order.
constexpr int kSumThreads = 128;

struct SumArgs {
    const uint2* tokens;
    RowsArg rows;
    FastDiv inner;
    char* table;
    int64_t pitch;
    float* partial;  // [chunks][2][width]
    uint32_t count, vocab, chunk, chunks;
    int width, threads;  // threads that share a row, a power of two
    float scale;
    int accumulate;
};

template <bool WIDE>
__device__ __forceinline__ int sum_column(int e, int t, int threads) {
    return WIDE ? t * 8 + e : e * threads + t;
}

// Eight columns of a row, from `first` on.
template <typename T, bool WIDE>
struct Piece {
    Raw8<T> raw;
    __device__ __forceinline__ void load(const char* row, int first, int t, int threads, int width) {
        raw = {};
        if (first + t * 8 < width) load8(raw, reinterpret_cast<const T*>(row) + first + t * 8);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const { unpack8(raw, x); }
};
template <typename T>
struct Piece<T, false> {
    T raw[8];
    __device__ __forceinline__ void load(const char* row, int first, int t, int threads, int width) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = first + sum_column<false>(e, t, threads);
            raw[e] = c < width ? reinterpret_cast<const T*>(row)[c] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_float(raw[e]);
    }
};

template <typename TO, bool WIDE>
__device__ __forceinline__ void write_row(const SumArgs& k, uint32_t id, const float (&sum)[8], int first, int t) {
    char* row = k.table + int64_t(id) * k.pitch;
    float x[8] = {};
    if (k.accumulate) {
        Piece<TO, WIDE> old;
        old.load(row, first, t, k.threads, k.width);
        old.get(x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += sum[e] * k.scale;
    if constexpr (WIDE) {
        if (first + t * 8 < k.width) store8(reinterpret_cast<TO*>(row) + first + t * 8, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = first + sum_column<false>(e, t, k.threads);
            if (c < k.width) reinterpret_cast<TO*>(row)[c] = from_float<TO>(x[e]);
        }
    }
}

template <typename TG, typename TO, bool WIDE>
__global__ void __launch_bounds__(kSumThreads) sum_tokens_kernel(const SumArgs k) {
    pdl_prologue();
    const int t = threadIdx.x % k.threads;
    const uint32_t chunk = blockIdx.x * (kSumThreads / k.threads) + threadIdx.x / k.threads;
    if (chunk >= k.chunks) return;
    const int first = blockIdx.y * (k.threads * 8);
    const uint32_t i0 = chunk * k.chunk, i1 = min(k.count, i0 + k.chunk);
    uint32_t id = __ldg(&k.tokens[i0]).x;
    if (id >= k.vocab) return;
    bool open = i0 > 0 && __ldg(&k.tokens[i0 - 1]).x == id;  // its tokens began in an earlier chunk
    const uint32_t next = i1 < k.count ? __ldg(&k.tokens[i1]).x : k.vocab;
    float sum[8] = {};
    auto leave = [&](int which) {
        float* to = k.partial + (int64_t(chunk) * 2 + which) * k.width + first;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = sum_column<WIDE>(e, t, k.threads);
            if (first + c < k.width) to[c] = sum[e];
        }
    };
    constexpr int U = 4;  // rows under way
    for (uint32_t i = i0; i < i1; i += U) {
        uint2 token[U];
        Piece<TG, WIDE> piece[U];
#pragma unroll
        for (int u = 0; u < U; ++u) token[u] = i + u < i1 ? __ldg(&k.tokens[i + u]) : make_uint2(k.vocab, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (token[u].x < k.vocab) piece[u].load(row_at(k.rows, k.inner, token[u].y), first, t, k.threads, k.width);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (token[u].x != id) {
                if (id < k.vocab) {
                    if (open) leave(0);
                    else write_row<TO, WIDE>(k, id, sum, first, t);
                }
                open = false;
                id = token[u].x;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] = 0.f;
            }
            if (id < k.vocab) {
                float x[8];
                piece[u].get(x);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += x[e];
            }
        }
    }
    if (id < k.vocab) {
        if (open) leave(0);
        else if (next == id) leave(1);
        else write_row<TO, WIDE>(k, id, sum, first, t);
    }
}

// One block for each chunk's end over which an id's tokens reach, where they begin in that chunk: 8 groups of threads take an eighth each of the chunks
// that follow, in order, and the eighths are added in order.
constexpr int kJoinGroups = 8;

template <typename TO, bool WIDE>
__global__ void __launch_bounds__(kSumThreads * kJoinGroups) join_kernel(const SumArgs k) {
    __shared__ float part[kJoinGroups][kSumThreads * 8];
    __shared__ uint32_t end;
    pdl_prologue();
    const uint32_t chunk = blockIdx.x;
    const uint32_t i1 = (chunk + 1) * k.chunk;  // (not the last chunk: the tokens go on)
    const uint32_t id = __ldg(&k.tokens[i1]).x;
    if (id >= k.vocab || __ldg(&k.tokens[i1 - 1]).x != id) return;
    const uint32_t i0 = chunk * k.chunk;
    if (i0 > 0 && __ldg(&k.tokens[i0]).x == id && __ldg(&k.tokens[i0 - 1]).x == id) return;  // they began earlier
    // the first chunk from the next one on that does not begin with the id
    if (threadIdx.x == 0) end = k.chunks;
    __syncthreads();
    for (uint32_t base = chunk + 1; base < k.chunks; base += blockDim.x) {
        const uint32_t c = base + threadIdx.x;
        if (c < k.chunks && __ldg(&k.tokens[c * k.chunk]).x != id) atomicMin(&end, c);
        __syncthreads();
        const bool found = end < k.chunks;
        __syncthreads();  // (before the next round's writes)
        if (found) break;
    }
    const uint32_t parts = end - chunk;  // [chunk][1], then [chunk + 1 ..][0]
    const int g = threadIdx.x / kSumThreads, t = threadIdx.x % kSumThreads;
    const uint32_t p0 = static_cast<uint32_t>(uint64_t(parts) * g / kJoinGroups), p1 = static_cast<uint32_t>(uint64_t(parts) * (g + 1) / kJoinGroups);
    for (int first = 0; first < k.width; first += kSumThreads * 8) {
        float sum[8] = {};
#pragma unroll 4
        for (uint32_t p = p0; p < p1; ++p) {
            const float* from = k.partial + (int64_t(chunk + p) * 2 + (p == 0 ? 1 : 0)) * k.width + first;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = e * kSumThreads + t;
                if (first + c < k.width) sum[e] += from[c];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) part[g][e * kSumThreads + t] = sum[e];
        __syncthreads();
        for (int c = threadIdx.x; c < kSumThreads * 8 && first + c < k.width; c += blockDim.x) {
            float total = part[0][c];
#pragma unroll
            for (int i = 1; i < kJoinGroups; ++i) total += part[i][c];
            TO* to = reinterpret_cast<TO*>(k.table + int64_t(id) * k.pitch) + first + c;
            const float x = total * k.scale + (k.accumulate ? to_float(*to) : 0.f);
            *to = from_float<TO>(x);
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

// How a gradient of many tokens is divided, and where its scratch lies.
struct Division {
    uint32_t chunk, chunks;
    int threads, tiles;
    int64_t token_bytes, partial_bytes;
    size_t bytes;
};

// Few tokens: rows owned by blocks, each of which reads all ids.  Many: sorted tokens.
constexpr int64_t kOwnedTokens = 512;

Division divide(const Problem& p) {
    Division d{};
    if (p.count <= kOwnedTokens || p.vocab == 0 || p.width == 0) return d;
    d.threads = 1;
    while (d.threads < kSumThreads && d.threads * 8 < p.width) d.threads *= 2;
    d.tiles = static_cast<int>(ceil_div(p.width, int64_t(d.threads) * 8));
    // chunks of 16 to 128 tokens: short ones where there are few tokens, so that each SM has eight chunks of whole rows; long ones leave fewer partial sums
    d.chunk = 16;
    while (d.chunk < 128 && p.count / d.chunk > int64_t(sm_count()) * 16) d.chunk *= 2;
    d.chunks = static_cast<uint32_t>(ceil_div(p.count, int64_t(d.chunk)));
    d.token_bytes = (p.count * 8 + 255) / 256 * 256;
    d.partial_bytes = (int64_t(d.chunks) * 2 * p.width * 4 + 255) / 256 * 256;
    d.bytes = static_cast<size_t>(2 * d.token_bytes + d.partial_bytes);
    return d;
}

void launch_owned_rows(b200_ctx* ctx, const b200_embedding_args& a, const Problem& p) {
    const int columns = static_cast<int>(std::min<int64_t>(p.width, kThreads * 4));
    const int64_t tiles = ceil_div(p.width, columns);
    // rows of sums: 40 KB at most (four blocks to an SM), and few enough that two blocks for each SM have some
    const int64_t most = std::min<int64_t>(1024, std::max<int64_t>(1, 10240 / columns));
    const int owned = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, ceil_div(p.vocab * tiles, sm_count() * 2))));
    const dim3 grid(static_cast<unsigned>(ceil_div(p.vocab, owned)), static_cast<unsigned>(tiles));
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

// The blocks of the sorting cluster: 16, where the device takes clusters that large, else 8.
int sort_cluster() {
    static int known[64] = {};
    int dev = 0;
    B200_CUDA_CHECK(cudaGetDevice(&dev));
    int& n = known[dev & 63];
    if (n == 0) {
        n = 8;
        if (cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = 16;
            cfg.blockDim = kSortThreads;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 16;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int fit = 0;
            if (cudaOccupancyMaxActiveClusters(&fit, sort_tokens_kernel, &cfg) == cudaSuccess && fit > 0) n = 16;
        }
        cudaGetLastError();
    }
    return n;
}

void launch_sorted(b200_ctx* ctx, const b200_embedding_args& a, const Problem& p, const Division& d) {
    char* scratch = operator_workspace(ctx, a.workspace, a.workspace_bytes, d.bytes);
    SortArgs s{};
    s.ids = p.ids;
    s.buffer[0] = reinterpret_cast<uint2*>(scratch);
    s.buffer[1] = reinterpret_cast<uint2*>(scratch + d.token_bytes);
    s.count = static_cast<uint32_t>(p.count);
    s.vocab = static_cast<uint32_t>(p.vocab);
    s.padding = a.padding_id < 0 ? INT64_MIN : a.padding_id;
    int bits = 1;
    while ((int64_t(1) << bits) <= p.vocab) ++bits;
    s.passes = (bits + 7) / 8;
    s.digit_bits = (bits + s.passes - 1) / s.passes;
    const bool accumulate = (a.flags & B200_ACCUMULATE) != 0;
    s.table = accumulate ? nullptr : static_cast<char*>(a.table.data);
    s.pitch = p.vocab > 1 ? p.pitch : p.width * static_cast<int64_t>(dtype_size(a.table.dtype));
    s.row_bytes = p.width * static_cast<int64_t>(dtype_size(a.table.dtype));
    s.status = ctx->d_status;
    const int cluster = sort_cluster();
    const unsigned clusters = accumulate ? 1u : static_cast<unsigned>(std::max(2, sm_count() * 2 / cluster));
    launch_kernel_clustered(ctx, sort_tokens_kernel, dim3(clusters * cluster), dim3(kSortThreads), 0, cluster, true, s);
    check_last_launch("embedding_backward");

    SumArgs k{};
    k.tokens = s.buffer[(s.passes + 1) & 1];
    k.rows = p.rows;
    k.inner = p.ids.inner;
    k.table = static_cast<char*>(a.table.data);
    k.pitch = p.pitch;
    k.partial = reinterpret_cast<float*>(scratch + 2 * d.token_bytes);
    k.count = s.count;
    k.vocab = s.vocab;
    k.chunk = d.chunk;
    k.chunks = d.chunks;
    k.width = static_cast<int>(p.width);
    k.threads = d.threads;
    k.scale = a.scale;
    k.accumulate = accumulate;
    const bool wide = p.width % 8 == 0 && aligned_rows(p.rows, 16) && reinterpret_cast<uintptr_t>(a.table.data) % 16 == 0 && p.pitch % 16 == 0;
    const dim3 grid(static_cast<unsigned>(ceil_div(int64_t(d.chunks) * d.threads, kSumThreads)), static_cast<unsigned>(d.tiles));
    with_types(a.table.dtype, a.rows.dtype, [&](auto to, auto tg) {
        using TO = decltype(to);
        using TG = decltype(tg);
        launch_kernel(ctx, wide ? sum_tokens_kernel<TG, TO, true> : sum_tokens_kernel<TG, TO, false>, grid, kSumThreads, 0, k);
        check_last_launch("embedding_backward");
        if (d.chunks > 1) launch_kernel(ctx, wide ? join_kernel<TO, true> : join_kernel<TO, false>, dim3(d.chunks - 1), kSumThreads * kJoinGroups, 0, k);
    });
    check_last_launch("embedding_backward");
    ctx->count_launch(d.chunks > 1 ? 3 : 2);
}

void launch_gradient(b200_ctx* ctx, const b200_embedding_args& a) {
    const Problem p = check_embedding(a, true);
    if (p.vocab == 0 || p.width == 0) return;
    if (p.width > int64_t(65535) * 1024) fail(B200_SHAPE_ERROR, "embedding_backward: a row of more than 65535 * 1024 elements");
    wait_for_tensors(ctx, {&a.table, &a.ids, &a.rows});
    ProfScope scope(ctx, "embedding_backward");
    const Division d = divide(p);
    if (d.bytes == 0) launch_owned_rows(ctx, a, p);
    else launch_sorted(ctx, a, p, d);
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
        *nbytes = divide(check_embedding(*args, true)).bytes;
    });
}

}  // extern "C"
