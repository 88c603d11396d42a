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

// Rows that start on a boundary of eight elements and hold whole eights: a thread moves kItems such pieces, kThreads pieces apart, so that their ids and then
// their elements are under way together.  (16384 rows of 1024, F32 to F16: 14.4 us with four pieces to a thread, 12.2 with two, 13.6 with one: four leave an SM
// half as many threads.)
constexpr int kItems = 2;

template <typename TI, typename TO>
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
}

// Other rows: a warp moves up to kStretch columns of a row, neighbours to neighbouring lanes.
constexpr int kStretch = 256;

template <typename TI, typename TO>
__global__ void __launch_bounds__(kThreads)
lookup_any_kernel(RowsArg out, const char* table, int64_t pitch, Ids ids, int64_t vocab, int64_t width, FastDiv stretches, int64_t total, float scale, uint32_t* status) {
    pdl_prologue();
    const int64_t task = int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    if (task >= total) return;
    const int lane = threadIdx.x % 32;
    uint32_t token, part;
    if (total < (int64_t(1) << 31)) {
        stretches.divmod(static_cast<uint32_t>(task), token, part);
    } else {
        token = static_cast<uint32_t>(task / stretches.d);
        part = static_cast<uint32_t>(task - int64_t(token) * stretches.d);
    }
    const int64_t id = ids[token];
    const bool in = id >= 0 && id < vocab;
    if (!in && lane == 0 && part == 0) atomicOr(status, kStatusIndexOutOfRange);
    const int64_t first = int64_t(part) * kStretch + lane;
    const TI* const from = reinterpret_cast<const TI*>(table + (in ? id : 0) * pitch) + first;
    TO* const to = reinterpret_cast<TO*>(row_at(out, ids.inner, token)) + first;
    TI raw[kStretch / 32];
#pragma unroll
    for (int k = 0; k < kStretch / 32; ++k) {
        if (in && first + k * 32 < width) raw[k] = from[k * 32];
    }
#pragma unroll
    for (int k = 0; k < kStretch / 32; ++k) {
        if (first + k * 32 < width) to[k * 32] = from_float<TO>(in ? to_float(raw[k]) * scale : 0.f);
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
                } else if ((id < 0 || (id >= vocab && id != padding)) && blockIdx.x == 0 && blockIdx.y == 0) {
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
            constexpr int kAtOnce = 16;  // rows under way: the most frequent ids' block has a good part of the tokens
            for (int j = 0; j < n; j += kAtOnce) {
                TG g[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    if (j + k < n) g[k] = reinterpret_cast<const TG*>(row_at(grad, ids.inner, list_token[j + k]))[col0 + c];
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    if (j + k < n) sums[int(list_row[j + k]) * columns + c] += to_float(g[k]);
                }
            }
        }
    }
    __syncthreads();
    // The rows side by side, each rounded up to a power of two of columns, so that narrow ones have all threads too.
    const int shift = cols > 1 ? 32 - __clz(cols - 1) : 0, cells = rows << shift;
    constexpr int kCells = 4;  // under way
    for (int first = tid; first < cells; first += kThreads * kCells) {
        float x[kCells] = {};
        if (accumulate) {
#pragma unroll
            for (int k = 0; k < kCells; ++k) {
                const int cell = first + k * kThreads, r = cell >> shift, c = cell & ((1 << shift) - 1);
                if (cell < cells && c < cols && (touched[r / 32] >> (r % 32) & 1)) x[k] = to_float(reinterpret_cast<const TO*>(table + (row0 + r) * pitch)[col0 + c]);
            }
        }
#pragma unroll
        for (int k = 0; k < kCells; ++k) {
            const int cell = first + k * kThreads, r = cell >> shift, c = cell & ((1 << shift) - 1);
            if (cell >= cells || c >= cols) continue;
            const bool any = touched[r / 32] >> (r % 32) & 1;
            if (any) x[k] += sums[r * columns + c] * scale;  // (else zeros whatever the scale)
            if (any || !accumulate) reinterpret_cast<TO*>(table + (row0 + r) * pitch)[col0 + c] = from_float<TO>(x[k]);
        }
    }
}

// ---- gradient: sorted tokens --------------------------------------------------

// The tokens are sorted by id, those of one id in their own order: radix passes over up to 8 bits of the id, of two kernels each.  A block has a tile of
// the tokens, a warp a stretch of the tile.  count_kernel leaves the counts of the tile's digits; move_kernel ranks every token among those of
// its digit in its stretch, adds the counts of the warps, the tiles and the digits before, and moves each token to its place.  Tokens that have no gradient
// sort behind all others, as id V.  The memory is idle meanwhile, so blocks behind those that sort write zeros over the table's last rows; the sums leave a
// bit for each row that has a token, and the rest of the rows without one is written at the end.  Up to 32768 tokens one cluster of blocks sorts in one launch (sort_cluster_kernel).
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMostHeld = 8;        // tokens of a thread of many blocks
constexpr int kMostClusterHeld = 2; // ... and of a cluster's: 131072 tokens by 16 blocks of 8 to a thread took 40 us, by 64 blocks 27
constexpr int kScannedTiles = 64;   // up to here move_kernel adds up the tiles' counts itself; above, scan_kernel does beforehand

// Rows of the table that are to be zeros.
struct Zeros {
    char* table;  // null: none
    int64_t pitch;
    uint32_t row0, rows;
    FastDiv pieces;  // of a row: of 16 bytes where `wide`, else of 2
    bool wide;
};

struct SortArgs {
    Ids ids;
    const uint2* from;   // (id, token); null: the ids
    uint2* to;
    uint32_t* counts;    // [tiles][256]; from scan_kernel, the counts of the tiles before
    uint32_t* totals;    // [256], from scan_kernel
    uint32_t* touched;   // a bit for each row, cleared here; or null
    uint32_t count, vocab, tiles, tile;  // tile: tokens of one
    int64_t padding;  // below 0: none, and no id is equal to it
    int shift, bits;
    bool scanned;
    Zeros zeros;
    uint32_t* status;
};

// Thread `tid` of `threads` writes its share of the zeros of 32 rows; `skip`: the rows that have a token.
__device__ __forceinline__ void zero_rows(const Zeros& z, uint32_t row0, uint32_t rows, uint32_t skip, uint32_t tid, uint32_t threads) {
    const uint32_t n = rows * z.pieces.d;  // (32 rows of less than 2^26 pieces)
    for (uint32_t i = tid; i < n; i += threads) {
        uint32_t r, c;
        z.pieces.divmod(i, r, c);
        if ((skip >> r) & 1) continue;
        char* to = z.table + int64_t(row0 + r) * z.pitch;
        if (z.wide) reinterpret_cast<uint4*>(to)[c] = make_uint4(0, 0, 0, 0);
        else reinterpret_cast<uint16_t*>(to)[c] = 0;
    }
}
// The blocks behind the tiles'.
__device__ __forceinline__ bool zeros_block(const SortArgs& k) {
    if (blockIdx.x < k.tiles) return false;
    for (uint32_t r = (blockIdx.x - k.tiles) * 32; r < k.zeros.rows; r += (gridDim.x - k.tiles) * 32) {
        zero_rows(k.zeros, k.zeros.row0 + r, min(32u, k.zeros.rows - r), 0, threadIdx.x, blockDim.x);
    }
    return true;
}

// Token i of a tile's thread, as (id, token).
__device__ __forceinline__ uint2 sort_token(const SortArgs& k, uint32_t i, bool report) {
    if (k.from != nullptr) return k.from[i];
    const int64_t id = k.ids[i];
    const bool in = id >= 0 && id < int64_t(k.vocab);
    if (report && !in && (id < 0 || id != k.padding)) atomicOr(k.status, kStatusIndexOutOfRange);
    return make_uint2(in && id != k.padding ? static_cast<uint32_t>(id) : k.vocab, i);
}

// The lanes that have the same digit (none: 256 and above), in nine votes.
__device__ __forceinline__ uint32_t same_digit(uint32_t d) {
    const uint32_t in = __ballot_sync(0xffffffffu, d < 256);
    uint32_t peers = d < 256 ? in : ~in;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const uint32_t ones = __ballot_sync(0xffffffffu, (d >> b) & 1);
        peers &= (d >> b) & 1 ? ones : ~ones;
    }
    return peers;
}

// HELD tokens of each thread, all under way at once: warp w has the 32 * HELD tokens from w * 32 * HELD on, 32 neighbours at a time.
template <int HELD>
__device__ __forceinline__ uint32_t held_index(const SortArgs& k, int h) {
    return blockIdx.x * k.tile + (threadIdx.x / 32 * HELD + h) * 32 + threadIdx.x % 32;
}

template <int HELD>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const SortArgs k) {
    __shared__ uint32_t counts[256];
    pdl_prologue();
    if (zeros_block(k)) return;
    if (k.touched != nullptr && k.from == nullptr) {
        for (uint32_t i = blockIdx.x * kSortThreads + threadIdx.x; i < (k.vocab + 31) / 32; i += k.tiles * kSortThreads) k.touched[i] = 0;
    }
    uint2 x[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const uint32_t i = held_index<HELD>(k, h);
        if (i < k.count) x[h] = sort_token(k, i, true);
    }
    if (threadIdx.x < 256) counts[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const bool in = held_index<HELD>(k, h) < k.count;
        const uint32_t d = in ? (x[h].x >> k.shift) & ((1u << k.bits) - 1) : 256u;
        const uint32_t peers = same_digit(d);  // (frequent tokens would queue up at one counter)
        if (in && threadIdx.x % 32 == __ffs(peers) - 1) atomicAdd(&counts[d], __popc(peers));
    }
    __syncthreads();
    if (threadIdx.x < 256) k.counts[blockIdx.x * 256 + threadIdx.x] = counts[threadIdx.x];
}

// A block to a digit: the tiles' counts become those of the tiles before, and their total.
__global__ void __launch_bounds__(kSortThreads) scan_kernel(const SortArgs k) {
    __shared__ uint32_t upto[kSortWarps];
    pdl_prologue();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint32_t before = 0;
    for (uint32_t base = 0; base < k.tiles; base += kSortThreads) {
        const uint32_t i = base + threadIdx.x;
        const uint32_t n = i < k.tiles ? k.counts[int64_t(i) * 256 + blockIdx.x] : 0;
        uint32_t scan = n;
#pragma unroll
        for (int s = 1; s < 32; s *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, scan, s);
            if (lane >= s) scan += other;
        }
        if (lane == 31) upto[warp] = scan;
        __syncthreads();
        uint32_t below = lane < warp ? upto[lane] : 0, all = upto[lane];
#pragma unroll
        for (int s = 16; s > 0; s /= 2) {
            below += __shfl_xor_sync(0xffffffffu, below, s);
            all += __shfl_xor_sync(0xffffffffu, all, s);
        }
        if (i < k.tiles) k.counts[int64_t(i) * 256 + blockIdx.x] = before + below + scan - n;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) k.totals[blockIdx.x] = before;
}

template <int HELD>
__global__ void __launch_bounds__(kSortThreads) move_kernel(const SortArgs k) {
    __shared__ uint32_t place[kSortWarps][257];  // counts of each warp's digits, then of the warps before; a row of odd length keeps columns off one bank
    __shared__ uint32_t base[256];               // where this tile's tokens of a digit go
    __shared__ uint32_t upto[kSortWarps];
    pdl_prologue();
    if (zeros_block(k)) return;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, d4 = tid / 4, q = tid % 4;
    uint2 x[HELD];
    uint32_t order[HELD];  // a token's rank among those of its digit in the stretch
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const uint32_t i = held_index<HELD>(k, h);
        if (i < k.count) x[h] = sort_token(k, i, false);
    }
    // the tiles before, and all: four threads to a digit
    uint32_t all = 0, before = 0;
    if (k.scanned) {
        all = q == 0 ? k.totals[d4] : 0;
        before = q == 0 ? k.counts[int64_t(blockIdx.x) * 256 + d4] : 0;
    } else {
        uint32_t n[kScannedTiles / 4];
#pragma unroll
        for (int i = 0; i < kScannedTiles / 4; ++i) n[i] = i * 4 + q < k.tiles ? k.counts[(i * 4 + q) * 256 + d4] : 0;
#pragma unroll
        for (int i = 0; i < kScannedTiles / 4; ++i) {
            all += n[i];
            if (i * 4 + q < blockIdx.x) before += n[i];
        }
    }
#pragma unroll
    for (int s = 1; s < 4; s *= 2) {
        all += __shfl_xor_sync(0xffffffffu, all, s);
        before += __shfl_xor_sync(0xffffffffu, before, s);
    }
    uint32_t scan = all;  // of the warp's 8 digits
#pragma unroll
    for (int s = 4; s < 32; s *= 2) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, scan, s);
        if (lane >= s) scan += other;
    }
    if (lane == 31) upto[warp] = scan;
    for (int i = lane; i < 257; i += 32) place[warp][i] = 0;
    __syncwarp();
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const bool in = held_index<HELD>(k, h) < k.count;
        const uint32_t d = in ? (x[h].x >> k.shift) & ((1u << k.bits) - 1) : 256u;
        const uint32_t peers = same_digit(d);
        const uint32_t sofar = place[warp][d];
        order[h] = sofar + __popc(peers & ((1u << lane) - 1));
        __syncwarp();
        if (lane == __ffs(peers) - 1) place[warp][d] = sofar + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    uint32_t below = lane < warp ? upto[lane] : 0;
#pragma unroll
    for (int s = 16; s > 0; s /= 2) below += __shfl_xor_sync(0xffffffffu, below, s);
    if (q == 0) base[d4] = below + scan - all + before;
    {  // exclusive over the warps: eight warps to a thread
        uint32_t n[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            n[i] = place[q * 8 + i][d4];
            sum += n[i];
        }
        uint32_t upper = sum;
#pragma unroll
        for (int s = 1; s < 4; s *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, upper, s, 4);
            if (q >= s) upper += other;
        }
        upper -= sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            place[q * 8 + i][d4] = upper;
            upper += n[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        if (held_index<HELD>(k, h) >= k.count) continue;
        const uint32_t d = (x[h].x >> k.shift) & ((1u << k.bits) - 1);
        k.to[base[d] + place[warp][d] + order[h]] = x[h];
    }
}

// The same sort by the blocks of one cluster, which hold all tokens: a pass reads the counts of the other blocks and moves the tokens through the cluster's
// shared memory.  One launch where the kernels above are four.
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
// Where the shared memory at `mine` lies in block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_address(const void* mine, uint32_t rank) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    return there;
}
__device__ __forceinline__ uint32_t cluster_load(uint32_t at) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ void cluster_store(uint32_t at, uint2 x) {
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(x.x), "r"(x.y) : "memory");
}
constexpr int kMostCluster = 16;

template <int HELD>
__global__ void __launch_bounds__(kSortThreads) sort_cluster_kernel(SortArgs k) {
    extern __shared__ uint2 held[];              // [kSortThreads * HELD]: this block's tokens between passes
    __shared__ uint32_t place[kSortWarps][257];  // (as in move_kernel)
    __shared__ uint32_t total[256], local[256], base[256], upto[kSortWarps];
    pdl_prologue();
    const uint32_t blocks = cluster_blocks(), rank = cluster_rank();
    k.tiles = blocks;  // (the first cluster's blocks are the tiles)
    if (zeros_block(k)) return;  // (whole clusters)
    constexpr uint32_t kTile = kSortThreads * HELD;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, d4 = tid / 4, q = tid % 4;
    if (k.touched != nullptr) {
        for (uint32_t i = rank * kSortThreads + tid; i < (k.vocab + 31) / 32; i += blocks * kSortThreads) k.touched[i] = 0;
    }
    uint2 x[HELD];
    uint32_t order[HELD];
    for (k.shift = 0; k.shift < 32 && (k.vocab >> k.shift) != 0; k.shift += k.bits) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const uint32_t i = held_index<HELD>(k, h);
            if (i < k.count) x[h] = k.shift == 0 ? sort_token(k, i, true) : held[i - rank * kTile];
        }
        for (int i = lane; i < 257; i += 32) place[warp][i] = 0;
        __syncwarp();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const bool in = held_index<HELD>(k, h) < k.count;
            const uint32_t d = in ? (x[h].x >> k.shift) & ((1u << k.bits) - 1) : 256u;
            const uint32_t peers = same_digit(d);
            const uint32_t sofar = place[warp][d];
            order[h] = sofar + __popc(peers & ((1u << lane) - 1));
            __syncwarp();
            if (lane == __ffs(peers) - 1) place[warp][d] = sofar + __popc(peers);
            __syncwarp();
        }
        __syncthreads();
        uint32_t mine = 0;  // this block's tokens of digit d4
        {  // exclusive over the warps
            uint32_t n[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[i] = place[q * 8 + i][d4];
                sum += n[i];
            }
            uint32_t upper = sum;
#pragma unroll
            for (int s = 1; s < 4; s *= 2) {
                const uint32_t other = __shfl_up_sync(0xffffffffu, upper, s, 4);
                if (q >= s) upper += other;
            }
            mine = __shfl_sync(0xffffffffu, upper, 3, 4);
            if (q == 0) total[d4] = mine;
            upper -= sum;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                place[q * 8 + i][d4] = upper;
                upper += n[i];
            }
        }
        // The digits before, among this block's tokens: these are put in order here first, so that neighbours move to the other blocks together.
        auto digits_before = [&](uint32_t n) {
            uint32_t scan = n;  // of the warp's 8 digits
#pragma unroll
            for (int s = 4; s < 32; s *= 2) {
                const uint32_t other = __shfl_up_sync(0xffffffffu, scan, s);
                if (lane >= s) scan += other;
            }
            if (lane == 31) upto[warp] = scan;
            __syncthreads();
            uint32_t below = lane < warp ? upto[lane] : 0;
#pragma unroll
            for (int s = 16; s > 0; s /= 2) below += __shfl_xor_sync(0xffffffffu, below, s);
            return below + scan - n;
        };
        const uint32_t here = digits_before(mine);
        if (q == 0) local[d4] = here;
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (held_index<HELD>(k, h) >= k.count) continue;
            const uint32_t d = (x[h].x >> k.shift) & ((1u << k.bits) - 1);
            held[local[d] + place[warp][d] + order[h]] = x[h];
        }
        __syncthreads();
        const uint32_t tokens = min(k.count, (rank + 1) * kTile) - min(k.count, rank * kTile);
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if (h * kSortThreads + tid < tokens) x[h] = held[h * kSortThreads + tid];
        }
        cluster_sync();  // the counts are there, and every block's tokens are in registers
        uint32_t n[kMostCluster / 4], all = 0, before = 0;
#pragma unroll
        for (int i = 0; i < kMostCluster / 4; ++i) n[i] = i * 4 + q < blocks ? cluster_load(cluster_address(&total[d4], i * 4 + q)) : 0;
#pragma unroll
        for (int i = 0; i < kMostCluster / 4; ++i) {
            all += n[i];
            if (i * 4 + q < rank) before += n[i];
        }
#pragma unroll
        for (int s = 1; s < 4; s *= 2) {
            all += __shfl_xor_sync(0xffffffffu, all, s);
            before += __shfl_xor_sync(0xffffffffu, before, s);
        }
        const uint32_t everywhere = digits_before(all);
        if (q == 0) base[d4] = everywhere + before - here;  // a token's place from its place in this block
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const uint32_t slot = h * kSortThreads + tid;
            if (slot >= tokens) continue;
            const uint32_t at = base[(x[h].x >> k.shift) & ((1u << k.bits) - 1)] + slot;
            cluster_store(cluster_address(&held[at % kTile], at / kTile), x[h]);
        }
        cluster_sync();  // the moved tokens are there, and no block reads another's counts any more
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const uint32_t slot = h * kSortThreads + tid, i = rank * kTile + slot;
        if (i < k.count) k.to[i] = held[slot];
    }
}

// The sorted tokens are cut into chunks of equal length, one to each group of threads that share a row.  A thread walks its chunk with a sum for each
// of its eight columns; where the id changes, the sum is that row of the table, unless the id's tokens reach over an end of the chunk.  Such sums meet in
// shared memory: the group where they begin adds up those of the groups behind it.  What reaches over an end of the block is left in `partial`,
// [block][0] where it began in an earlier block, [block][1] where it begins here, and join_kernel adds those up.  Always in the tokens' order.
constexpr int kSumThreads = 256;

struct SumArgs {
    const uint2* tokens;
    uint32_t* touched;   // a bit for each row that has a token; null: not wanted
    RowsArg rows;
    FastDiv inner;
    char* table;
    int64_t pitch;
    float* partial;  // [blocks][2][width]
    uint32_t count, vocab, chunk, blocks;  // blocks: along the tokens
    int width, threads, tiles;  // threads that share a row, a power of two up to 128; tiles of threads * 8 columns
    float scale;
    int accumulate;
    uint32_t join_blocks, zero_words;  // join_kernel's blocks; groups of 32 rows to each of its blocks behind those
    Zeros zeros;
};

// Once for each row that has a token.
__device__ __forceinline__ void mark_row(const SumArgs& k, uint32_t id, int first, int t) {
    if (k.touched != nullptr && first == 0 && t == 0) atomicOr(&k.touched[id / 32], 1u << (id % 32));
}

template <typename TO, bool WIDE>
__device__ __forceinline__ void write_row(const SumArgs& k, uint32_t id, const float (&sum)[8], int first, int t) {
    char* row = k.table + int64_t(id) * k.pitch;
    mark_row(k, id, first, t);
    float x[8] = {};
    if (k.accumulate) {
        Piece<TO, WIDE> old;
        old.load(row, first, t, k.threads, k.width);
        old.get(x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += sum[e] * k.scale;
    store_piece<TO, WIDE>(row, x, first, t, k.threads, k.width);
}

template <typename TG, typename TO, bool WIDE>
__global__ void __launch_bounds__(kSumThreads, 2) sum_tokens_kernel(const SumArgs k) {
    __shared__ float meet[2][8][kSumThreads];  // sums that reach over a chunk's end: [began earlier, begins here][column][thread]
    // of each group: the id of its first and last token (V: none), and which sums it left: 1: began earlier, 2: begins here, 4: the first goes on behind the chunk
    __shared__ uint32_t left[kSumThreads], first_id[kSumThreads], last_id[kSumThreads];
    pdl_prologue();
    const uint32_t block = blockIdx.x / k.tiles;
    const int first = static_cast<int>(blockIdx.x % k.tiles) * (k.threads * 8);
    const int groups = kSumThreads / k.threads, group = threadIdx.x / k.threads, t = threadIdx.x % k.threads;
    const uint32_t chunk = block * groups + group;
    const uint32_t i0 = min(k.count, chunk * k.chunk), i1 = min(k.count, i0 + k.chunk);
    uint32_t id = k.vocab, marks = 0, start = k.vocab;
    if (i0 < i1) {
        start = id = __ldg(&k.tokens[i0]).x;
        const uint32_t before = i0 > 0 ? __ldg(&k.tokens[i0 - 1]).x : k.vocab, next = i1 < k.count ? __ldg(&k.tokens[i1]).x : k.vocab;
        bool open = id < k.vocab && before == id;  // its tokens began in an earlier chunk
        float sum[8] = {};
        auto leave = [&](int which) {
            marks |= 1u << which;
#pragma unroll
            for (int e = 0; e < 8; ++e) meet[which][e][threadIdx.x] = sum[e];
        };
        constexpr int U = WIDE ? 8 : 4;  // rows under way, and the tokens behind them
        uint2 token[U], next_token[U];
#pragma unroll
        for (int u = 0; u < U; ++u) next_token[u] = i0 + u < i1 ? __ldg(&k.tokens[i0 + u]) : make_uint2(k.vocab, 0);
        for (uint32_t i = i0; i < i1 && id < k.vocab; i += U) {
            Piece<TG, WIDE> piece[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                token[u] = next_token[u];
                if (token[u].x < k.vocab) piece[u].load(row_at(k.rows, k.inner, token[u].y), first, t, k.threads, k.width);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) next_token[u] = i + U + u < i1 ? __ldg(&k.tokens[i + U + u]) : make_uint2(k.vocab, 0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u >= i1) break;
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
            if (open) {
                leave(0);
                if (next == id) marks |= 4;
            } else if (next == id) {
                leave(1);
            } else {
                write_row<TO, WIDE>(k, id, sum, first, t);
            }
        }
    }
    if (t == 0) left[group] = marks, first_id[group] = start, last_id[group] = id;
    __syncthreads();
    // Sums that begin in this block, and the one that the block's first group continues from the block before.
    for (int which = 1; which >= 0; --which) {
        const bool mine = which == 1 ? (left[group] & 2) != 0 : group == 0 && (left[0] & 1) != 0;
        if (!mine) continue;
        float sum[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = meet[which][e][threadIdx.x];
        bool on = which == 1 || (left[0] & 4) != 0;  // goes on into the next group
        int g = group + 1;
        for (; on && g < groups; ++g) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += meet[0][e][g * k.threads + t];
            on = (left[g] & 4) != 0;
        }
        const uint32_t of = which == 1 ? last_id[group] : first_id[0];
        if (which == 0 || on) {  // over an end of the block
            if (which == 1) mark_row(k, of, first, t);
            float* to = k.partial + (int64_t(block) * 2 + which) * k.width + first;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = piece_column<WIDE>(e, t, k.threads);
                if (first + c < k.width) to[c] = sum[e];
            }
        } else {
            write_row<TO, WIDE>(k, of, sum, first, t);
        }
    }
}

// One block for each end of a block of sums that an id's tokens reach over, where they begin in that block, and each kJoinColumns columns: four groups of
// threads take a quarter each of the partial sums, in order, and the quarters are added in order.  Few of these blocks have something to do, and that
// waits more than it moves; so the zeros of rows without a token are written by blocks behind them.
constexpr int kJoinColumns = 256, kJoinThreads = kJoinColumns / 4, kJoinGroups = 4;

template <typename TO>
__global__ void __launch_bounds__(kJoinThreads * kJoinGroups) join_kernel(const SumArgs k) {
    __shared__ float part[kJoinGroups][kJoinColumns];
    __shared__ uint32_t end;
    pdl_prologue();
    if (blockIdx.x >= k.join_blocks) {
        const uint32_t word0 = (blockIdx.x - k.join_blocks) * k.zero_words;
        for (uint32_t w = word0; w < word0 + k.zero_words && w * 32 < k.zeros.rows; ++w) {
            zero_rows(k.zeros, w * 32, min(32u, k.zeros.rows - w * 32), __ldg(&k.touched[w]), threadIdx.x, kJoinThreads * kJoinGroups);
        }
        return;
    }
    const uint32_t span = k.chunk * (kSumThreads / k.threads);  // tokens of a block
    const int column_blocks = (k.width + kJoinColumns - 1) / kJoinColumns;
    const uint32_t block = blockIdx.x / column_blocks, i0 = block * span, i1 = i0 + span;  // (not the last block: the tokens go on)
    const uint32_t before = i0 > 0 ? __ldg(&k.tokens[i0 - 1]).x : k.vocab, begin = __ldg(&k.tokens[i0]).x, last = __ldg(&k.tokens[i1 - 1]).x, id = __ldg(&k.tokens[i1]).x;
    if (threadIdx.x == 0) end = k.blocks;
    if (id >= k.vocab || last != id || (begin == id && before == id)) return;  // nothing over the end, or it began earlier
    __syncthreads();
    // the first block from the next one on that does not begin with the id
    for (uint32_t from = block + 1; from < k.blocks; from += blockDim.x) {
        const uint32_t c = from + threadIdx.x;
        if (c < k.blocks && __ldg(&k.tokens[c * span]).x != id) atomicMin(&end, c);
        __syncthreads();
        const bool found = end < k.blocks;
        __syncthreads();  // (before the next round's writes)
        if (found) break;
    }
    const uint32_t parts = end - block;  // [block][1], then [block + 1 ..][0]
    const int g = threadIdx.x / kJoinThreads, t = threadIdx.x % kJoinThreads;
    const uint32_t p0 = static_cast<uint32_t>(uint64_t(parts) * g / kJoinGroups), p1 = static_cast<uint32_t>(uint64_t(parts) * (g + 1) / kJoinGroups);
    const int first = static_cast<int>(blockIdx.x % column_blocks) * kJoinColumns;
    float sum[4] = {};
#pragma unroll 8
    for (uint32_t p = p0; p < p1; ++p) {
        const float* from = k.partial + (int64_t(block + p) * 2 + (p == 0 ? 1 : 0)) * k.width + first;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = e * kJoinThreads + t;
            if (first + c < k.width) sum[e] += from[c];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[g][e * kJoinThreads + t] = sum[e];
    __syncthreads();
    const int c = threadIdx.x;
    if (first + c < k.width) {
        float total = part[0][c];
#pragma unroll
        for (int i = 1; i < kJoinGroups; ++i) total += part[i][c];
        TO* to = reinterpret_cast<TO*>(k.table + int64_t(id) * k.pitch) + first + c;
        const float x = total * k.scale + (k.accumulate ? to_float(*to) : 0.f);
        *to = from_float<TO>(x);
    }
}

struct Problem {
    int64_t count, vocab, width, pitch;
    Ids ids;
    RowsArg rows;
    bool wide;               // rows and table hold whole eights on their boundaries
    int64_t pieces, blocks;  // of a lookup: pieces of a row, and blocks of all of them
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
    p.wide = p.width % 8 == 0 && aligned_rows(p.rows, a.rows.dtype) && aligned_rows(RowsArg{static_cast<char*>(a.table.data), 0, p.pitch}, a.table.dtype);
    p.pieces = p.wide ? p.width / 8 : ceil_div(p.width, kStretch);
    p.blocks = ceil_div(p.count * p.pieces, p.wide ? kThreads * kItems : kThreads / 32);
    if (!backward && p.blocks >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "embedding: too many elements");
    if (backward && p.vocab != 0 && p.width >= int64_t(1) << 24) fail(B200_SHAPE_ERROR, "embedding_backward: a row of 2^24 elements or more");
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
    ProfScope scope(ctx, "embedding");
    const char* table = static_cast<const char*>(a.table.data);
    const FastDiv by(static_cast<uint32_t>(p.pieces));
    const int64_t total = p.count * p.pieces;
    with_types(a.table.dtype, a.rows.dtype, [&](auto ti, auto to) {
        using TI = decltype(ti);
        using TO = decltype(to);
        const dim3 grid(static_cast<unsigned>(p.blocks));
        if (p.wide) launch_kernel(ctx, lookup_kernel<TI, TO>, grid, kThreads, 0, p.rows, table, p.pitch, p.ids, p.vocab, by, total, a.scale, ctx->d_status);
        else launch_kernel(ctx, lookup_any_kernel<TI, TO>, grid, kThreads, 0, p.rows, table, p.pitch, p.ids, p.vocab, p.width, by, total, a.scale, ctx->d_status);
    });
    check_last_launch("embedding");
    ctx->count_launch();
}

using SortCluster = void (*)(SortArgs);
SortCluster sort_cluster(int held) {
    return held == 1 ? sort_cluster_kernel<1> : sort_cluster_kernel<2>;
}

// How many clusters of `blocks` blocks the current device holds at once; 0 where it takes none of them.
int clusters_at_once(int held, int blocks) {
    static std::mutex mutex;
    static int known[64][2][5] = {};  // device, held, blocks: one more than the answer
    int dev = 0, h = 0, b = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return blocks <= 8 ? 1 : 0;
    }
    while ((1 << h) < held) ++h;
    while ((1 << b) < blocks) ++b;
    std::lock_guard<std::mutex> lock(mutex);
    int& n = known[dev & 63][h][b];
    if (n == 0) {
        const size_t shared = static_cast<size_t>(kSortThreads) * held * sizeof(uint2);
        int fit = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = static_cast<unsigned>(blocks);
        cfg.blockDim = kSortThreads;
        cfg.dynamicSmemBytes = shared;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(blocks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const SortCluster kernel = sort_cluster(held);
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)) != cudaSuccess ||
            (blocks > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
            cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;  // (not kept: the question failed, not the device)
        }
        n = fit + 1;
    }
    return n - 1;
}
int largest_cluster() { return clusters_at_once(kMostClusterHeld, kMostCluster) > 0 ? kMostCluster : 8; }

// How a gradient of many tokens is divided, and where its scratch lies.
struct Division {
    uint32_t chunk, blocks;
    int threads, tiles;
    int held;             // (from choose_sort) tokens of a thread that sorts
    int cluster;          // blocks of the cluster that sorts; 0: many blocks
    uint32_t sort_tiles;
    int64_t token_bytes, touched_bytes, partial_bytes, count_bytes;
    size_t bytes;
};

// Few tokens and no large table, or a small one: rows owned by blocks, each of which reads all ids.  Else sorted tokens, whose launches take 12 to 14 us together, beside which
// zeros are written.  (F32, owned and sorted: 128 tokens of 1000 x 64 5.5 us and 12.3, 512 tokens 13.5 and 13.7; of 1000 x 512 9.7 and 14.4, 27.6 and 14.4; 8 tokens
// of 50000 x 128 13.9 and 12.3, of 50000 x 1024 77.8 and 41.2.)
bool is_owned(int64_t count, int64_t elements) { return (count <= 128 && elements <= 1 << 22) || (count <= 512 && elements <= 1 << 17); }

constexpr int64_t kMostClusterTokens = int64_t(kSortThreads) * kMostClusterHeld * kMostCluster;

// Tokens of a thread where many blocks sort: few tiles, as every block adds up the counts of all; but eight at most.
int tokens_held(int64_t count) {
    int held = 1;
    while (held < kMostHeld && ceil_div(count, int64_t(kSortThreads) * held) > kScannedTiles) held *= 2;
    return held;
}

Division divide(const Problem& p) {
    Division d{};
    if (p.vocab == 0 || p.width == 0 || p.count == 0 || is_owned(p.count, p.vocab * p.width)) return d;
    d.threads = 1;
    while (d.threads < 128 && d.threads * 8 < p.width) d.threads *= 2;
    d.tiles = static_cast<int>(ceil_div(p.width, int64_t(d.threads) * 8));
    const int groups = kSumThreads / d.threads;
    // two waves of blocks, two to an SM, of chunks that are no longer than 256 tokens
    const int64_t wave = std::max<int64_t>(1, int64_t(sm_count()) * 4 / d.tiles);
    d.chunk = static_cast<uint32_t>(std::min<int64_t>(256, std::max<int64_t>(4, ceil_div(ceil_div(p.count, wave * groups), 4) * 4)));
    d.blocks = static_cast<uint32_t>(ceil_div(ceil_div(p.count, int64_t(d.chunk)), groups));
    auto whole = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    d.token_bytes = whole(p.count * 8);
    d.touched_bytes = whole(ceil_div(p.vocab, 32) * 4);
    d.partial_bytes = whole(int64_t(d.blocks) * 2 * p.width * 4);
    // As many tiles as any way to sort asks for, whatever clusters the device takes.
    const int64_t most_tiles = p.count <= kMostClusterTokens ? ceil_div(p.count, kSortThreads) : ceil_div(p.count, int64_t(kSortThreads) * tokens_held(p.count));
    d.count_bytes = most_tiles * 1024 + 1024;
    d.bytes = static_cast<size_t>(2 * d.token_bytes + d.touched_bytes + d.partial_bytes + d.count_bytes);
    return d;
}

// Who sorts: asks the device for its clusters.
void choose_sort(Division& d, const Problem& p) {
    if (d.bytes == 0) return;
    d.held = 1;
    const int most = p.count <= kMostClusterTokens ? largest_cluster() : 0;
    if (p.count <= int64_t(kSortThreads) * kMostClusterHeld * most) {
        // as few tokens to a thread as the cluster allows; a smaller cluster where one token is enough
        while (int64_t(kSortThreads) * d.held * most < p.count) d.held *= 2;
        d.cluster = 1;
        while (int64_t(kSortThreads) * d.held * d.cluster < p.count) d.cluster *= 2;
    } else {
        d.held = tokens_held(p.count);
    }
    d.sort_tiles = static_cast<uint32_t>(ceil_div(p.count, int64_t(kSortThreads) * d.held));
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
                      static_cast<uint32_t>(p.count), p.vocab, p.width, owned, columns, a.padding_id, a.scale,
                      static_cast<int>(a.flags & B200_ACCUMULATE), ctx->d_status);
    });
    check_last_launch("embedding_backward");
    ctx->count_launch();
}

// Zeros written beside the sort: what the memory takes meanwhile, of one kernel of the many and of the cluster's.
constexpr int64_t kZerosBesideKernel = int64_t(20) << 20, kZerosBesideCluster = int64_t(48) << 20;

void launch_sorted(b200_ctx* ctx, const b200_embedding_args& a, const Problem& p, const Division& d, char* scratch) {
    const bool accumulate = (a.flags & B200_ACCUMULATE) != 0;
    const int64_t size = static_cast<int64_t>(dtype_size(a.table.dtype)), row_bytes = p.width * size;
    uint2* buffer[2] = {reinterpret_cast<uint2*>(scratch), reinterpret_cast<uint2*>(scratch + d.token_bytes)};
    scratch += 2 * d.token_bytes;
    SortArgs s{};
    s.ids = p.ids;
    s.touched = accumulate ? nullptr : reinterpret_cast<uint32_t*>(scratch);
    scratch += d.touched_bytes;
    float* partial = reinterpret_cast<float*>(scratch);
    scratch += d.partial_bytes;
    s.totals = reinterpret_cast<uint32_t*>(scratch);
    s.counts = s.totals + 256;
    s.count = static_cast<uint32_t>(p.count);
    s.vocab = static_cast<uint32_t>(p.vocab);
    s.padding = a.padding_id;
    s.tiles = d.sort_tiles;
    s.tile = static_cast<uint32_t>(kSortThreads * d.held);
    s.scanned = d.sort_tiles > kScannedTiles;
    s.status = ctx->d_status;
    int bits = 1;
    while ((int64_t(1) << bits) <= p.vocab) ++bits;
    const int passes = (bits + 7) / 8;
    s.bits = (bits + passes - 1) / passes;
    Zeros zeros{};
    uint32_t zeros_left = 0;  // rows, from the first on, whose zeros are not written yet
    int64_t early = 0;        // rows beside each kernel of the sort
    if (!accumulate) {
        zeros.table = static_cast<char*>(a.table.data);
        zeros.pitch = p.pitch;
        zeros.wide = ((reinterpret_cast<uintptr_t>(zeros.table) | static_cast<uintptr_t>(p.pitch) | static_cast<uintptr_t>(row_bytes)) & 15) == 0;
        zeros.pieces = FastDiv(static_cast<uint32_t>(row_bytes / (zeros.wide ? 16 : 2)));
        zeros_left = s.vocab;
        early = (d.cluster > 0 ? kZerosBesideCluster : kZerosBesideKernel) / row_bytes / 32 * 32;
    }
    auto take_zeros = [&] {
        s.zeros = zeros;
        s.zeros.row0 = static_cast<uint32_t>(zeros_left > early ? (zeros_left - early + 31) / 32 * 32 : 0);
        s.zeros.rows = zeros_left > s.zeros.row0 ? zeros_left - s.zeros.row0 : 0;
        zeros_left -= s.zeros.rows;
        return static_cast<unsigned>(std::min<int64_t>(sm_count() * 2, ceil_div(int64_t(s.zeros.rows), 32)));
    };
    auto sort = [&](auto kernel) {
        const unsigned beside = take_zeros();
        launch_kernel(ctx, kernel, dim3(s.tiles + beside), kSortThreads, 0, s);
        check_last_launch("embedding_backward");
        ctx->count_launch();
    };
    if (d.cluster > 0) {
        s.to = buffer[0];
        const int at_once = clusters_at_once(d.held, d.cluster);
        if (at_once < 1) fail(B200_DEVICE_ERROR, "embedding_backward: the device takes no cluster of " + std::to_string(d.cluster) + " blocks");
        const unsigned beside = static_cast<unsigned>(std::min<int64_t>(std::max(1, at_once - 1), ceil_div(int64_t(take_zeros()), d.cluster)));
        launch_kernel_clustered(ctx, sort_cluster(d.held), dim3((1 + beside) * d.cluster), dim3(kSortThreads), static_cast<size_t>(kSortThreads) * d.held * sizeof(uint2), d.cluster, false, s);  // (not early: clusters of 16 wait for a GPC's SMs, which a kernel before may hold)
        check_last_launch("embedding_backward");
        ctx->count_launch();
    }
    for (int pass = 0; pass < passes && d.cluster == 0; ++pass) {
        s.from = pass == 0 ? nullptr : buffer[(pass + 1) & 1];
        s.to = buffer[pass & 1];
        s.shift = pass * s.bits;
        sort(d.held == 1 ? count_kernel<1> : d.held == 2 ? count_kernel<2> : d.held == 4 ? count_kernel<4> : count_kernel<8>);
        if (s.scanned) {
            launch_kernel(ctx, scan_kernel, dim3(256), kSortThreads, 0, s);
            check_last_launch("embedding_backward");
            ctx->count_launch();
        }
        sort(d.held == 1 ? move_kernel<1> : d.held == 2 ? move_kernel<2> : d.held == 4 ? move_kernel<4> : move_kernel<8>);
    }
    SumArgs k{};
    k.tokens = s.to;
    k.touched = s.touched;
    k.rows = p.rows;
    k.inner = p.ids.inner;
    k.table = static_cast<char*>(a.table.data);
    k.pitch = p.pitch;
    k.partial = partial;
    k.count = s.count;
    k.vocab = s.vocab;
    k.chunk = d.chunk;
    k.blocks = d.blocks;
    k.width = static_cast<int>(p.width);
    k.threads = d.threads;
    k.tiles = d.tiles;
    k.scale = a.scale;
    k.accumulate = accumulate;
    k.zeros = zeros;
    k.zeros.rows = zeros_left;
    k.zero_words = static_cast<uint32_t>(std::max<int64_t>(1, (128 << 10) / (32 * row_bytes)));
    k.join_blocks = static_cast<uint32_t>((d.blocks - 1) * ceil_div(p.width, kJoinColumns));
    const uint32_t last_blocks = k.join_blocks + static_cast<uint32_t>(ceil_div(ceil_div(int64_t(zeros_left), 32), int64_t(k.zero_words)));
    with_types(a.table.dtype, a.rows.dtype, [&](auto to, auto tg) {
        using TO = decltype(to);
        using TG = decltype(tg);
        launch_kernel(ctx, p.wide ? sum_tokens_kernel<TG, TO, true> : sum_tokens_kernel<TG, TO, false>, dim3(d.blocks * static_cast<uint32_t>(d.tiles)), kSumThreads, 0, k);
        check_last_launch("embedding_backward");
        if (last_blocks > 0) launch_kernel(ctx, join_kernel<TO>, dim3(last_blocks), kJoinThreads * kJoinGroups, 0, k);
    });
    check_last_launch("embedding_backward");
    ctx->count_launch(last_blocks > 0 ? 2 : 1);
}

void launch_gradient(b200_ctx* ctx, const b200_embedding_args& a) {
    const Problem p = check_embedding(a, true);
    if (p.vocab == 0 || p.width == 0) return;
    Division d = divide(p);
    check_workspace(a.workspace, a.workspace_bytes, d.bytes);
    choose_sort(d, p);
    char* const scratch = operator_workspace(ctx, a.workspace, d.bytes);  // (refuses, too, before anything is queued)
    wait_for_tensors(ctx, {&a.table, &a.ids, &a.rows});
    ProfScope scope(ctx, "embedding_backward");
    if (d.bytes == 0) launch_owned_rows(ctx, a, p);
    else launch_sorted(ctx, a, p, d, scratch);
}

}  // namespace

void check_embedding_call(const b200_embedding_args& a, bool backward) {
    const Problem p = check_embedding(a, backward);
    if (backward && a.workspace != nullptr) check_workspace(a.workspace, a.workspace_bytes, divide(p).bytes);
}

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
