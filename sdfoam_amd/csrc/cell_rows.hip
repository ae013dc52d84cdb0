// Rows of a per-cell table (features, embeddings) for a list of cells, and the
// gradients of the table and the weights.
//
//   rows[i, :]       = scale w_i table[c_i, :]          (0 where c_i is no cell)
//   table_grad[v, :] = sum over { i : c_i = v } of scale w_i rows_grad[i, :]
//   weight_grad[i]   = scale <table[c_i, :], rows_grad[i, :]>
//
// The table's gradient is formed cell by cell from the ids in sorted order
// (stable, so a cell's rows are added in the order of their positions): no sum
// depends on the order of atomics, every run gives the same bits.  Sums are
// held in fp32 and rounded to the table's type once.
#include "label_device.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;

namespace {

// A row in pieces of kP elements, one to a lane: 16 bytes, or single elements
// for rows shorter than that.  A last piece that would pass the row's end lies
// where it ends there: two lanes then hold one element, of the same value.
template <typename T, int kP> struct Piece {
    T v[kP];
};
template <typename T, int kP> __device__ __forceinline__ Piece<T, kP> load_piece(const T *p) {
    Piece<T, kP> c;
    __builtin_memcpy(&c, p, sizeof(c));
    return c;
}
template <typename T, int kP>
__device__ __forceinline__ void store_piece(T *p, const Piece<T, kP> &c) {
    __builtin_memcpy(p, &c, sizeof(c));
}
// Read or written once: past the caches (single elements: as above).
template <typename T, int kP> __device__ __forceinline__ Piece<T, kP> load_piece_past(const T *p) {
    if constexpr (sizeof(Piece<T, kP>) == 16) return load_past<Piece<T, kP>, sizeof(T)>(p);
    else return load_piece<T, kP>(p);
}
template <typename T, int kP>
__device__ __forceinline__ void store_piece_past(T *p, const Piece<T, kP> &c) {
    if constexpr (sizeof(c) == 16) store_past<sizeof(T)>(p, c);
    else store_piece<T, kP>(p, c);
}
template <int kP> __device__ __forceinline__ uint32_t column(uint32_t piece, uint32_t width) {
    return min(piece * kP, width - kP);
}

// t / d for t d < 2^32, by the reciprocal `m` = 2^32 / d rounded up (d > 1)
struct Divisor {
    uint32_t d, m;
};
__device__ __forceinline__ uint32_t operator/(uint32_t t, Divisor d) {
    return d.d == 1 ? t : __umulhi(t, d.m);
}
Divisor divisor(uint32_t d) { return {d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }

constexpr uint32_t kXcds = 8;
// Blocks go to the XCDs in turn; neighbouring rows often share cells, so each
// XCD takes a run of blocks and keeps their table rows in its own L2.
__device__ __forceinline__ uint64_t block_of_xcd(uint32_t b, uint32_t blocks) {
    const uint32_t each = blocks / kXcds, whole = each * kXcds;
    return b < whole ? (b % kXcds) * each + b / kXcds : b;
}

// ---- the rows ------------------------------------------------------------------

struct RowsArgs {
    const void *table;
    uint64_t stride;
    uint32_t num_cells, width;
    Divisor pieces; // of a row
    const void *cells;
    int id_type;
    uint64_t first, count; // rows of this launch
    uint32_t per;          // rows a block
    const float *weight;
    float scale;
    void *rows;
};

constexpr int kUnroll = 4;
constexpr uint64_t kWindow = 1ull << 18; // blocks a launch: it holds fewer than 2^32 threads
constexpr uint32_t kMaxWidth = 1u << 18; // of a row: Divisor's range

// One lane per piece of a row, kUnroll of them in flight: bound by the bytes of
// the rows read and written (the ids come once per row, from L1 after that).
// 1.92M rows of 49 floats, 460 MB: 77 to 109 us; 8 pieces in flight a lane or 2
// are slower (165, 142 against 136 before the writes went past the caches).
template <typename T, int kP, bool kPast>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
    const T *table = static_cast<const T *>(a.table);
    T *out = static_cast<T *>(a.rows);
    const uint64_t r0 = a.first + block_of_xcd(blockIdx.x, gridDim.x) * a.per;
    const uint32_t rows = (uint32_t)min((uint64_t)a.per, a.first + a.count - r0);
    const uint32_t items = rows * a.pieces.d;
    for (uint32_t t = threadIdx.x; t < items; t += 256u * kUnroll) {
        int32_t cell[kUnroll];
        uint32_t row[kUnroll], col[kUnroll];
        float f[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t k = min(t + u * 256u, items - 1);
            row[u] = k / a.pieces;
            col[u] = column<kP>(k - row[u] * a.pieces.d, a.width);
            cell[u] = load_id(a.cells, a.id_type, r0 + row[u], a.num_cells);
            f[u] = a.weight ? a.scale * a.weight[r0 + row[u]] : a.scale;
        }
        Piece<T, kP> p[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (cell[u] >= 0)
                p[u] = load_piece<T, kP>(table + (uint64_t)cell[u] * a.stride + col[u]);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (t + u * 256u >= items) continue;
            Piece<T, kP> o;
#pragma unroll
            for (int e = 0; e < kP; ++e) o.v[e] = (T)(cell[u] < 0 ? 0.0f : f[u] * (float)p[u].v[e]);
            T *to = out + (r0 + row[u]) * a.width + col[u];
            if constexpr (kPast) store_piece_past<T, kP>(to, o);
            else store_piece<T, kP>(to, o);
        }
    }
}

// ---- the sort of the ids: stable, least significant digit first ---------------

constexpr uint32_t kSortThreads = 1024;
constexpr uint32_t kSortWaves = kSortThreads / 64;
constexpr uint32_t kSteps = 4;                       // keys per thread
constexpr uint32_t kTile = kSteps * kSortThreads;    // keys of one block
// One block sorts up to a tile alone, and up to kOneBlock keys where the clearing
// beside it takes as long.  Several blocks for one there: 6,000 ids in 1M cells of 49
// floats 62 -> 50 us, 12,000 in 1M of 64 71 -> 66, 16,384 in 2M of 64 108 -> 100; rows
// of 2,048 halves, 8,000 ids in 65,536 cells 94 -> 88, 16,381 98 -> 92, but 16,384 in
// 65,429 85 -> 89; beside 134 MB, below the limit, 10,000 64 -> 64, 16,384 69 -> 75.
constexpr uint32_t kOneBlock = 16 * kSortThreads;
constexpr uint64_t kOneBlockClears = 192ull << 20;
constexpr uint32_t kMaxBits = 11;                    // of a digit
constexpr uint32_t kFewTilesBits = 10;               // where tiles are few
constexpr uint32_t kScanParts = 16;                  // threads that share a digit's tiles
// Up to so many tiles, each tile's block adds up the counts of all tiles itself, a
// digit per thread, for the scan's launch (100,000 cells: 32,000 ids 37 -> 35 us,
// 131,072 43 -> 38, 500,000 59 -> 60; 2M cells in three passes of 7 bits for two of
// 11 with their scans: 262,144 ids 64 -> 59, 1M 97 -> 103).
constexpr uint32_t kFewTiles = 64;

// The table's gradient is cleared by extra blocks of the sort's launches, which
// leave the memory idle: each launch clears [begin, end) of it, `each` bytes a
// block in stores of 16, past the caches (which would otherwise be full of
// zeros when the sums begin: 120 -> 96 us for 268 MB).  Few large shares: beside
// the sort's blocks a CU has room (LDS) for one of these at a time.
struct Clear {
    char *to;
    uint64_t begin, end, each;
};
constexpr uint32_t kClearStep = kSortThreads * 16 * 4;
constexpr uint32_t kClearBlocks = 512;
__device__ __forceinline__ void clear_block(const Clear &c, uint32_t block) {
    const uint64_t begin = c.begin + block * c.each;
    const uint64_t end = begin + c.each < c.end ? begin + c.each : c.end;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (uint64_t base = begin; base < end; base += kClearStep) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint64_t at = base + (k * kSortThreads + threadIdx.x) * 16ull;
            if (at + 16 <= end) store_past<2>(c.to + at, zero);
            else
                for (uint64_t b = at; b < end; ++b) c.to[b] = 0;
        }
    }
}

struct SortPass {
    const void *ids; // first pass: the caller's ids; NULL: `in`
    int id_type;
    uint32_t num_cells;
    const uint2 *in; // {key, position}
    uint2 *out;
    // the ids' factors move with them: gathered by position, each would cost a
    // line of memory
    const float *weight; // the caller's, in the first pass times `scale`; NULL: none
    float scale;
    float *weight_out;
    uint32_t *counts; // [tiles][digits], after the scan those of the tiles before
    uint32_t *totals; // [digits]
    uint32_t n, tiles, shift, bits, passes;
    bool scanned;    // counts and totals; else counts as they were made, and no totals
    uint32_t blocks; // those after them clear
    Clear clear;
};

// no cell sorts last
__device__ __forceinline__ uint2 sort_item(const SortPass &p, uint32_t i) {
    if (!p.ids) return p.in[i];
    const int32_t c = load_id(p.ids, p.id_type, i, p.num_cells);
    return make_uint2(c < 0 ? p.num_cells : (uint32_t)c, i);
}

// How often each digit occurs in each tile (1M ids: 7 us, with its share of the
// clearing, as is the scan).
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortPass p) {
    extern __shared__ uint32_t hist[];
    if (blockIdx.x >= p.blocks) return clear_block(p.clear, blockIdx.x - p.blocks);
    const uint32_t digits = 1u << p.bits;
    const uint32_t base = blockIdx.x * kTile;
    uint32_t key[kSteps];
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r) {
        const uint32_t i = base + r * kSortThreads + threadIdx.x;
        key[r] = i < p.n ? sort_item(p, i).x : 0u;
    }
    for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r)
        if (base + r * kSortThreads + threadIdx.x < p.n)
            atomicAdd(&hist[(key[r] >> p.shift) & (digits - 1)], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads)
        p.counts[(uint64_t)blockIdx.x * digits + d] = hist[d];
}

// Per digit, the exclusive sums over the tiles and the total: 64 digits a
// block, kScanParts threads each with a run of tiles.
__global__ __launch_bounds__(64 * kScanParts) void sort_scan_kernel(SortPass p) {
    __shared__ uint32_t sums[kScanParts][64];
    if (blockIdx.x >= p.blocks) return clear_block(p.clear, blockIdx.x - p.blocks);
    const uint32_t digits = 1u << p.bits;
    const uint32_t d = blockIdx.x * 64u + (threadIdx.x & 63u), part = threadIdx.x >> 6;
    const uint32_t each = (p.tiles + kScanParts - 1) / kScanParts;
    const uint32_t lo = min(part * each, p.tiles), hi = min(lo + each, p.tiles);
    uint32_t s = 0;
    if (d < digits)
#pragma unroll 8
        for (uint32_t t = lo; t < hi; ++t) s += p.counts[(uint64_t)t * digits + d];
    sums[part][threadIdx.x & 63u] = s;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (uint32_t k = 0; k < kScanParts; ++k) {
        const uint32_t v = sums[k][threadIdx.x & 63u];
        if (k < part) before += v;
        total += v;
    }
    if (d >= digits) return;
    if (part == 0) p.totals[d] = total;
#pragma unroll 8
    for (uint32_t t = lo; t < hi; ++t) {
        const uint32_t v = p.counts[(uint64_t)t * digits + d];
        p.counts[(uint64_t)t * digits + d] = before;
        before += v;
    }
}

// One tile's items, and what a block needs of LDS to put them in order by a
// digit: counters per wavefront and digit, and in their place the items.
template <uint32_t kSteps> struct Tile {
    uint2 item[kSteps];
    float f[kSteps];
};
unsigned order_bytes(uint32_t bits, size_t item_bytes) {
    const size_t counters = kSortWaves * sizeof(uint16_t) << bits;
    return (unsigned)((sizeof(uint32_t) << bits) + (counters > item_bytes ? counters : item_bytes));
}

// Orders a tile of `count` items by the digit at p.shift, stably, into LDS
// (kFactors: and their factors behind them).  Thread t has items (t / 64) * 64
// kSteps + r * 64 + t % 64.  Each wavefront ranks its own: the lanes of equal
// digits find each other by one ballot per bit, and the wavefront's counter of
// the digit carries the rank from one step of 64 to the next.  to_output: also
// shift[digit], from a place in the tile to one in the whole output.
template <bool kFactors, uint32_t kSteps>
__device__ __forceinline__ uint2 *order_tile(const SortPass &p, Tile<kSteps> &x, uint32_t count,
                                             bool to_output, uint32_t *shift, uint2 *waves) {
    const uint32_t digits = 1u << p.bits;
    uint16_t *seen = reinterpret_cast<uint16_t *>(shift + digits); // [kSortWaves][digits]
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    const uint32_t base = w * (kSteps * 64);
    constexpr uint32_t kEach = (1u << kMaxBits) / kSortThreads; // digits per thread at most
    const uint32_t each = (digits + kSortThreads - 1) / kSortThreads, lo = threadIdx.x * each;
    uint32_t total[kEach], earlier[kEach], here[kEach], rank[kSteps];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        const bool has = to_output && k < each && lo + k < digits;
        total[k] = has && p.scanned ? p.totals[lo + k] : 0u;
        earlier[k] = has && p.scanned ? p.counts[(uint64_t)blockIdx.x * digits + lo + k] : 0u;
    }
    if (to_output && !p.scanned && lo < digits) { // one digit per thread then
        const uint32_t *counts = p.counts + lo;
#pragma unroll 16
        for (uint32_t t = 0; t < p.tiles; ++t) {
            const uint32_t c = counts[(uint64_t)t * digits];
            total[0] += c;
            earlier[0] += t < blockIdx.x ? c : 0u;
        }
    }
    uint16_t *own = seen + w * digits;
    for (uint32_t d = lane; d < digits; d += 64u) own[d] = 0;
    wave_sync();
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r) {
        const bool in = base + r * 64u + lane < count;
        const uint32_t d = (x.item[r].x >> p.shift) & (digits - 1);
        uint64_t same = __ballot(in);
        for (uint32_t b = 0; b < p.bits; ++b) {
            const uint64_t set = __ballot((d >> b) & 1u);
            same &= (d >> b) & 1u ? set : ~set;
        }
        const uint32_t below = __popcll(same & ((1ull << lane) - 1ull));
        const uint32_t so_far = own[d];
        rank[r] = so_far + below;
        wave_sync(); // every lane has read before the first of each digit adds
        if (in && below == 0) own[d] = (uint16_t)(so_far + (uint32_t)__popcll(same));
        wave_sync();
    }
    __syncthreads();
    // where each digit starts: in the output (x) and in this tile (y)
    uint2 mine = make_uint2(0u, 0u);
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        here[k] = 0;
        if (k < each && lo + k < digits)
            for (uint32_t v = 0; v < kSortWaves; ++v) here[k] += seen[v * digits + lo + k];
        mine.x += total[k];
        mine.y += here[k];
    }
    uint2 s = mine;
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t a = __shfl_up(s.x, d), b = __shfl_up(s.y, d);
        if (lane >= d) s.x += a, s.y += b;
    }
    if (lane == 63u) waves[w] = s;
    __syncthreads();
    uint32_t out = s.x - mine.x, in_tile = s.y - mine.y;
    for (uint32_t k = 0; k < w; ++k) out += waves[k].x, in_tile += waves[k].y;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        if (k >= each || lo + k >= digits) break;
        shift[lo + k] = out + earlier[k] - in_tile;
        uint32_t at = in_tile;
        for (uint32_t v = 0; v < kSortWaves; ++v) {
            uint16_t &c = seen[v * digits + lo + k];
            const uint32_t was = c;
            c = (uint16_t)at;
            at += was;
        }
        out += total[k];
        in_tile += here[k];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r)
        rank[r] += own[(x.item[r].x >> p.shift) & (digits - 1)];
    __syncthreads(); // the items take the counters' place
    uint2 *tile = reinterpret_cast<uint2 *>(seen);
    float *factor = reinterpret_cast<float *>(tile + kSteps * kSortThreads);
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r)
        if (base + r * 64u + lane < count) {
            tile[rank[r]] = x.item[r];
            if (kFactors && p.weight) factor[rank[r]] = x.f[r];
        }
    __syncthreads();
    return tile;
}
template <bool kFactors, uint32_t kSteps>
__device__ __forceinline__ void load_tile(const SortPass &p, uint32_t begin, Tile<kSteps> &x) {
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r) {
        const uint32_t i = begin + (threadIdx.x >> 6) * (kSteps * 64) + r * 64u + (threadIdx.x & 63u);
        x.item[r] = i < p.n ? sort_item(p, i) : make_uint2(0u, 0u);
        x.f[r] = kFactors && p.weight && i < p.n ? p.scale * p.weight[i] : 0.0f;
    }
}

// Puts a tile in order and writes it from LDS: lanes side by side then write
// side by side (1M ids with factors, 10-bit digits: 16 us, 22 without; 19 with a
// share of the clearing).  Bound by the pieces of lines it writes: tiles of 8,192
// would write longer ones, but on half the CUs (22 us).
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortPass p) {
    extern __shared__ uint32_t shift[];
    __shared__ uint2 waves[kSortWaves];
    if (blockIdx.x >= p.blocks) return clear_block(p.clear, blockIdx.x - p.blocks);
    const uint32_t begin = blockIdx.x * kTile, count = min(kTile, p.n - begin);
    Tile<kSteps> x;
    load_tile<true>(p, begin, x);
    const uint2 *tile = order_tile<true>(p, x, count, true, shift, waves);
    const float *factor = reinterpret_cast<const float *>(tile + kTile);
#pragma unroll
    for (uint32_t r = 0; r < kSteps; ++r) {
        const uint32_t k = r * kSortThreads + threadIdx.x;
        if (k >= count) break;
        const uint2 y = tile[k];
        const uint32_t to = k + shift[(y.x >> p.shift) & ((1u << p.bits) - 1)];
        p.out[to] = y;
        if (p.weight) p.weight_out[to] = factor[k];
    }
}

// At most kSteps * kSortThreads ids: every pass in one block, without leaving
// LDS.  The factors stay where they are: so few are read by position from L2.
// 16,381 ids: 35 us alone, 50 beside the clearing of 268 MB; 4,096: 11.
template <uint32_t kSteps>
__global__ __launch_bounds__(kSortThreads) void sort_block_kernel(SortPass p) {
    extern __shared__ uint32_t shift[];
    __shared__ uint2 waves[kSortWaves];
    if (blockIdx.x >= p.blocks) return clear_block(p.clear, blockIdx.x - p.blocks);
    Tile<kSteps> x;
    load_tile<false>(p, 0, x);
    const uint2 *tile = nullptr;
    for (uint32_t k = 0; k < p.passes; ++k) {
        if (k > 0) {
#pragma unroll
            for (uint32_t r = 0; r < kSteps; ++r) {
                const uint32_t i =
                    (threadIdx.x >> 6) * (kSteps * 64) + r * 64u + (threadIdx.x & 63u);
                if (i < p.n) x.item[r] = tile[i];
            }
            __syncthreads();
        }
        p.shift = k * p.bits;
        tile = order_tile<false>(p, x, p.n, false, shift, waves);
    }
    for (uint32_t k = threadIdx.x; k < p.n; k += kSortThreads) p.out[k] = tile[k];
}

// ---- the sums -------------------------------------------------------------------

// The sorted ids in tiles of `tile` positions, a tile to kLanes lanes (which
// hold a row, or 64 pieces of it).  A cell whose positions all lie in one tile
// is summed and written there.  Of a cell that goes on in other tiles, each
// tile keeps its sum in fp32: slot 0 where the cell began in an earlier tile,
// slot 1 where it begins here; join_rows_kernel adds them.
// Bound by the bytes: 1M rows of 64 bfloat16 in 300,000 cells, weights'
// gradient beside: 68 us for about 300 MB (111 when each id's weight was
// gathered by its position); 16,381 rows of 2,048 halves: 28.
struct SumsArgs {
    const void *grad;
    uint64_t stride;
    uint32_t width, num_cells;
    const uint2 *order; // {cell, position} of the ids, sorted by cell
    uint32_t n, tile, tiles;
    const float *factor; // scale and weight in the order of `order`; NULL:
    const float *weight; // the caller's (NULL: 1), times scale
    float scale;
    float *partial; // [tiles][2][width]
    void *table_grad;
    const void *table; // with weight_grad
    uint64_t table_stride;
    float *weight_grad; // NULL: not formed here
};

constexpr int kBatch = 4; // rows in flight per lane (8: 100 VGPRs, half the waves, 167 us for 117)

template <typename T, int kP, int kLanes>
__device__ __forceinline__ void sum_tile(const SumsArgs &a, uint32_t tile, uint32_t piece, uint32_t l) {
    const T *grad = static_cast<const T *>(a.grad);
    T *out = static_cast<T *>(a.table_grad);
    const bool mine = piece * kP < a.width; // lanes past the row hold nothing
    const uint32_t col = mine ? column<kP>(piece, a.width) : 0u;
    const uint32_t p0 = tile * a.tile, p1 = min(p0 + a.tile, a.n);
    const uint32_t before = p0 > 0 ? a.order[p0 - 1].x : a.num_cells;
    const uint32_t after = p1 < a.n ? a.order[p1].x : a.num_cells;
    float acc[kP] = {};
    uint32_t cell = a.order[p0].x;
    bool open = cell == before; // the first cell began in an earlier tile
    const auto flush = [&](bool goes_on) {
        if (!mine || cell >= a.num_cells) return;
        if (open || goes_on) {
            float *to = a.partial + ((uint64_t)tile * 2 + (open ? 0 : 1)) * a.width + col;
#pragma unroll
            for (int e = 0; e < kP; ++e) to[e] = acc[e];
        } else {
            Piece<T, kP> o;
#pragma unroll
            for (int e = 0; e < kP; ++e) o.v[e] = (T)acc[e];
            store_piece<T, kP>(out + (uint64_t)cell * a.width + col, o);
        }
    };
    for (uint32_t p = p0; p < p1; p += kBatch) {
        uint32_t key[kBatch], index[kBatch];
        float f[kBatch];
        Piece<T, kP> g[kBatch], t[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const uint2 id = a.order[min(p + b, p1 - 1)];
            key[b] = id.x;
            index[b] = id.y;
            f[b] = a.factor ? a.factor[min(p + b, p1 - 1)] : a.scale;
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const bool live = p + b < p1 && key[b] < a.num_cells;
            if (a.weight && !a.factor) f[b] *= a.weight[index[b]];
            f[b] = live ? f[b] : 0.0f;
            g[b] = {};
            if (live && mine) g[b] = load_piece_past<T, kP>(grad + (uint64_t)index[b] * a.stride + col);
            if (a.weight_grad) {
                t[b] = {};
                if (live && mine)
                    t[b] = load_piece<T, kP>(static_cast<const T *>(a.table) +
                                             (uint64_t)key[b] * a.table_stride + col);
            }
        }
        if (a.weight_grad) {
            // elements that two lanes hold count for the first of them
            const uint32_t own = mine ? piece * kP - col : 0u;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < kP; ++e)
                    if ((uint32_t)e >= own) s = fmaf((float)g[b].v[e], (float)t[b].v[e], s);
                s = group_sum<kLanes>(s);
                if (l == b % kLanes && p + b < p1) // (no cell: 0 whatever the scale)
                    a.weight_grad[index[b]] = key[b] < a.num_cells ? a.scale * s : 0.0f;
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (p + b >= p1) break;
            if (key[b] != cell) {
                flush(false);
                cell = key[b];
                open = false;
#pragma unroll
                for (int e = 0; e < kP; ++e) acc[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < kP; ++e) acc[e] = fmaf(f[b], (float)g[b].v[e], acc[e]);
        }
    }
    flush(cell == after);
}

template <typename T, int kP, int kLanes>
__global__ __launch_bounds__(256) void sums_kernel(SumsArgs a) {
    const uint32_t tile = (blockIdx.x * 256u + threadIdx.x) / kLanes, l = threadIdx.x % kLanes;
    if (tile < a.tiles) sum_tile<T, kP, kLanes>(a, tile, blockIdx.y * kLanes + l, l);
}

// The cells that go on past the tile they begin in: their tiles' sums in order.
// A group of lanes looks at the tiles that follow its own, one a lane (16 at
// least) and on to 64 while all are that cell's; where it goes on past those, the
// whole block adds its sums, every group a share of the tiles.  Bound by latency:
// 9 us for 1M rows of 64, 12 for 16,381 of 2,048, one cell of them in 125 tiles.
// (Blocks for all that pass 16 tiles: the gradient of 262,144 rows of 8 in 2,000
// cells 158 us for 43, of 200,000 rows of 32 in 100 cells 30 for 33.)
template <typename T, int kP, int kLanes>
__global__ __launch_bounds__(256) void join_rows_kernel(SumsArgs a) {
    constexpr uint32_t kGroups = 256 / kLanes;
    constexpr uint32_t kProbes = kLanes < 16 ? 16 / kLanes : 1, kRound = kProbes * kLanes;
    constexpr uint32_t kNear = 64;
    __shared__ uint32_t list[kGroups];
    __shared__ uint32_t listed;
    __shared__ float sums[4][kLanes * kP]; // of the wavefronts
    const uint32_t g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
    const uint32_t tile = blockIdx.x * kGroups + g, piece = blockIdx.y * kLanes + l;
    const bool mine = piece * kP < a.width;
    const uint32_t col = mine ? column<kP>(piece, a.width) : 0u;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const auto goes_on = [&](uint32_t t, uint32_t cell) {
        return t < a.tiles && a.order[(uint64_t)t * a.tile].x == cell;
    };
    // s += the sums of `count` tiles from `first` on, `step` apart
    const auto add = [&](float *s, uint32_t first, uint32_t count, uint32_t step) {
        for (uint32_t k = 0; k < count; k += 8) {
            float x[8][kP];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t t = first + min(k + u, count - 1) * step;
                __builtin_memcpy(x[u], a.partial + (uint64_t)t * 2 * a.width + col, sizeof(x[u]));
            }
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u)
                if (k + u < count)
#pragma unroll
                    for (int e = 0; e < kP; ++e) s[e] += x[u][e];
        }
    };
    const auto begun = [&](float *s, uint32_t t) {
        __builtin_memcpy(s, a.partial + ((uint64_t)t * 2 + 1) * a.width + col, kP * sizeof(float));
    };
    const auto write = [&](uint32_t cell, const float *s) {
        if (!mine) return;
        Piece<T, kP> o;
#pragma unroll
        for (int e = 0; e < kP; ++e) o.v[e] = (T)s[e];
        store_piece<T, kP>(static_cast<T *>(a.table_grad) + (uint64_t)cell * a.width + col, o);
    };
    if (tile + 1 < a.tiles) {
        const uint32_t p0 = tile * a.tile, cell = a.order[p0 + a.tile - 1].x;
        const bool whole = p0 > 0 && a.order[p0 - 1].x == cell; // the tile is all of that cell
        uint32_t near = 0; // the following tiles that begin with it: the first so many
        if (cell < a.num_cells && !whole) {
            for (uint32_t k = 0; k < kNear && near == k; k += kRound) {
                uint32_t n = 0;
#pragma unroll
                for (uint32_t q = 0; q < kProbes; ++q)
                    n += goes_on(tile + 1 + k + q * kLanes + l, cell);
                near += group_all<kLanes>(n, [](uint32_t x, uint32_t y) { return x + y; });
            }
        }
        if (near == kNear) {
            if (l == 0) list[atomicAdd(&listed, 1u)] = tile;
        } else if (near > 0) {
            float s[kP];
            begun(s, tile);
            add(s, tile + 1, near, 1);
            write(cell, s);
        }
    }
    __syncthreads();
    const uint32_t n = listed; // the order of the list does not matter: each has its own cell
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t first = list[i] + 1, cell = a.order[(uint64_t)first * a.tile].x;
        // the tiles that begin with it, counted by 256 probes at a time
        uint32_t lo = 0, range = a.tiles - first;
        while (range > 0) {
            const uint32_t step = (range + 255u) / 256u;
            const uint32_t at = lo + threadIdx.x * step;
            const uint32_t c = __syncthreads_count(threadIdx.x * step < range && goes_on(first + at, cell));
            if (step == 1) {
                lo += c;
                break;
            }
            // the last probe that met it is `lo`; from there on, fewer than step
            lo += (c - 1) * step;
            range = min(step, range - (c - 1) * step);
        }
        float s[kP] = {};
        if (g < lo) add(s, first + g, (lo - g + kGroups - 1) / kGroups, kGroups);
        // the wavefront's groups, then the wavefronts
#pragma unroll
        for (int e = 0; e < kP; ++e) {
#pragma unroll
            for (int d = kLanes; d < 64; d *= 2) s[e] += __shfl_xor(s[e], d);
            if ((threadIdx.x & 63u) < (uint32_t)kLanes) sums[threadIdx.x >> 6][l * kP + e] = s[e];
        }
        __syncthreads();
        if (g == 0) {
            begun(s, first - 1);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < kP; ++e) s[e] += sums[k][l * kP + e];
            write(cell, s);
        }
        __syncthreads();
    }
}

// The weights' gradient by itself, where the table's is not wanted or a row is
// wider than a wavefront holds: kLanes lanes an id, kUnroll ids at a time.  Bound
// by the two rows that each id reads (1M ids, rows of 64 bfloat16, 268 MB: 56
// us; a wavefront per id took 280).
template <typename T, int kP, int kLanes>
__global__ __launch_bounds__(256) void weight_grad_kernel(RowsArgs a, const T *__restrict__ grad,
                                                          uint64_t grad_stride,
                                                          float *__restrict__ weight_grad) {
    const uint32_t l = threadIdx.x % kLanes;
    const uint64_t first =
        a.first + ((uint64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes) * kUnroll;
    const uint64_t end = a.first + a.count;
    if (first >= end) return; // a whole group
    int32_t cell[kUnroll];
    float s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint64_t i = first + u < end ? first + u : end - 1;
        cell[u] = load_id(a.cells, a.id_type, i, a.num_cells);
        s[u] = 0.0f;
    }
    for (uint32_t k = l; k < a.pieces.d; k += kLanes) {
        const uint32_t col = column<kP>(k, a.width);
        Piece<T, kP> x[kUnroll], y[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            x[u] = {};
            y[u] = {};
            if (cell[u] < 0 || first + u >= end) continue;
            x[u] = load_piece_past<T, kP>(grad + (first + u) * grad_stride + col);
            y[u] = load_piece<T, kP>(static_cast<const T *>(a.table) + (uint64_t)cell[u] * a.stride + col);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int e = 0; e < kP; ++e) // elements that two lanes hold count once
                if (col + e >= k * kP) s[u] = fmaf((float)x[u].v[e], (float)y[u].v[e], s[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const float sum = group_sum<kLanes>(s[u]);
        if (l == u % kLanes && first + u < end) // (no cell: 0 whatever the scale)
            weight_grad[first + u] = cell[u] < 0 ? 0.0f : a.scale * sum;
    }
}

// ---- which kernel --------------------------------------------------------------

size_t align256(size_t x) { return (x + 255u) & ~(size_t)255u; }

template <int kV> struct Int {
    static constexpr int v = kV;
};
// f(element, elements of a piece) as types
template <typename F> void with_piece(int type, uint32_t width, F f) {
    with_type(type, [&](auto t) {
        constexpr int kP = 16 / (int)sizeof(t);
        if (width >= (uint32_t)kP) f(t, Int<kP>());
        else f(t, Int<1>());
    });
}
template <typename F> void with_lanes(uint32_t pieces, F f) {
    if (pieces <= 1) f(Int<1>());
    else if (pieces <= 2) f(Int<2>());
    else if (pieces <= 4) f(Int<4>());
    else if (pieces <= 8) f(Int<8>());
    else if (pieces <= 16) f(Int<16>());
    else if (pieces <= 32) f(Int<32>());
    else f(Int<64>());
}
uint32_t pieces_of(int type, uint32_t width) {
    const uint32_t p = 16 / (uint32_t)type_bytes(type);
    return width >= p ? (width + p - 1) / p : width;
}

// Positions a tile: as many as leave about 4,096 wavefronts, 8 at least.  (More
// positions a tile mean fewer sums to join.)
uint32_t tile_of(uint64_t count, uint32_t pieces) {
    uint32_t lanes = 1;
    while (lanes < pieces && lanes < 64) lanes *= 2;
    const uint64_t waves = count * lanes / 64 * ((pieces + lanes - 1) / lanes);
    uint32_t tile = 8;
    while (tile < 64 && waves / (tile * 2) >= 4096) tile *= 2;
    return tile;
}

struct Sort {
    uint32_t passes, bits, tiles;
    bool scan;
};
Sort sort_of(uint64_t num_cells, uint64_t count) {
    uint32_t bits = 1; // of the largest key, num_cells
    while ((num_cells >> bits) != 0) ++bits;
    Sort s;
    s.tiles = (uint32_t)((count + kTile - 1) / kTile);
    s.scan = s.tiles > kFewTiles;
    const uint32_t most = s.scan ? kMaxBits : kFewTilesBits;
    s.passes = (bits + most - 1) / most;
    s.bits = (bits + s.passes - 1) / s.passes;
    return s;
}

struct Layout {
    size_t order[2], factor[2], counts, totals, partial, bytes;
};
Layout layout_of(int type_size, uint64_t num_cells, uint32_t width, uint64_t count) {
    const uint32_t p = 16 / type_size;
    const uint32_t pieces = width >= p ? (width + p - 1) / p : width;
    const Sort s = sort_of(num_cells, count);
    const uint32_t tile = tile_of(count, pieces);
    const uint64_t tiles = (count + tile - 1) / tile;
    Layout o;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t was = at;
        at += align256(bytes);
        return was;
    };
    for (size_t &order : o.order) order = take(8 * count);
    for (size_t &factor : o.factor) factor = take(4 * count);
    o.counts = take(4ull * s.tiles << s.bits);
    o.totals = take(4ull << s.bits);
    o.partial = take(tiles * 2 * width * 4);
    o.bytes = at + 256;
    return o;
}

int check_rows(const char *what, int type, uint64_t num_cells, uint32_t width, int id_type,
               uint64_t count) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: unknown element type %d", what, type);
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "%s: unknown id type %d", what, id_type);
    if (num_cells >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 cells", what);
    if (count >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 ids", what);
    if (width > kMaxWidth)
        return fail(SDF_E_INVALID, "%s takes rows of at most 2^18 elements", what);
    return SDF_OK;
}

bool misaligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

} // namespace

extern "C" {

int sdf_cell_rows(int type, const void *table, uint64_t table_stride, uint64_t num_cells,
                  uint32_t width, int id_type, const void *cells, uint64_t count,
                  const float *weight, float scale, void *rows, void *stream) {
    const int rc = check_rows("cell_rows", type, num_cells, width, id_type, count);
    if (rc != SDF_OK) return rc;
    if (count == 0 || width == 0) return SDF_OK;
    if (!cells || !rows || (num_cells > 0 && !table))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    if (misaligned(table, type_bytes(type)) || misaligned(rows, type_bytes(type)))
        return fail(SDF_E_INVALID, "cell_rows: table and rows must be aligned to their elements");
    const uint32_t pieces = pieces_of(type, width);
    RowsArgs a = {table, table_stride, (uint32_t)num_cells, width, divisor(pieces), cells, id_type,
                  0, count, 1, weight, scale, rows};
    // Rows that no cache would keep for their reader are written past them
    // (1.92M rows of 49 floats, 376 MB: 135 -> 98 us; 1M of 64 bfloat16, 134 MB:
    // 51 -> 44; 16,384 of 2,048 halves, 67 MB: 23.9 and 24.4).
    const bool past = count * width * type_bytes(type) >= 128ull << 20;
    // 1,024 pieces a block, or 256 where that leaves CUs without one
    const uint64_t items = count * pieces < 1024 * 1024 ? 256 : 1024;
    a.per = (uint32_t)(items / pieces > 0 ? items / pieces : 1);
    with_piece(type, width, [&](auto t, auto p) {
        for (uint64_t r = 0; r < count; r += kWindow * a.per) {
            a.first = r;
            a.count = count - r < kWindow * a.per ? count - r : kWindow * a.per;
            const dim3 grid((unsigned)((a.count + a.per - 1) / a.per));
            hipStream_t s = static_cast<hipStream_t>(stream);
            using T = decltype(t);
            constexpr int kP = decltype(p)::v;
            if (past) hipLaunchKernelGGL((rows_kernel<T, kP, true>), grid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((rows_kernel<T, kP, false>), grid, dim3(256), 0, s, a);
        }
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "cell_rows");
}

size_t sdf_cell_rows_backward_scratch_bytes(uint64_t num_cells, uint32_t width, uint64_t count) {
    const size_t two = layout_of(2, num_cells, width, count).bytes;
    const size_t four = layout_of(4, num_cells, width, count).bytes;
    return two > four ? two : four;
}

int sdf_cell_rows_backward(int type, const void *rows_grad, uint64_t rows_grad_stride,
                           const void *table, uint64_t table_stride, uint64_t num_cells,
                           uint32_t width, int id_type, const void *cells, uint64_t count,
                           const float *weight, float scale, void *table_grad, float *weight_grad,
                           void *scratch, size_t scratch_bytes, void *stream) {
    const int rc = check_rows("cell_rows_backward", type, num_cells, width, id_type, count);
    if (rc != SDF_OK) return rc;
    if (!table_grad && !weight_grad) return SDF_OK;
    if ((count > 0 && !cells) ||
        (count > 0 && width > 0 && !rows_grad) || (table_grad && !scratch) ||
        (weight_grad && num_cells > 0 && width > 0 && !table))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    // (the weights' gradient by itself needs no scratch)
    const size_t need =
        table_grad ? sdf_cell_rows_backward_scratch_bytes(num_cells, width, count) : 0;
    if (scratch_bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    const size_t e_size = type_bytes(type);
    if (misaligned(rows_grad, e_size) || misaligned(table, e_size) || misaligned(table_grad, e_size))
        return fail(SDF_E_INVALID,
                    "cell_rows_backward: rows and tables must be aligned to their elements");
    if (table_grad && misaligned(scratch, 256)) return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t n = (uint32_t)count, cells_n = (uint32_t)num_cells;
    const uint32_t pieces = pieces_of(type, width);
    const bool sum = table_grad && num_cells > 0 && width > 0;
    // the weights' gradient beside the sums, where a group of lanes sees whole rows
    const bool beside = sum && weight_grad && pieces <= 64;
    char *at = static_cast<char *>(scratch);
    const Layout lay = layout_of((int)type_bytes(type), num_cells, width, count);
    SumsArgs a = {};
    if (sum) {
        // the launches of the sort clear the gradient between them
        const Sort so = sort_of(num_cells, count);
        const uint64_t bytes = num_cells * width * type_bytes(type);
        const bool alone = n <= kTile || (n <= kOneBlock && bytes >= kOneBlockClears);
        const uint32_t launches = alone ? 1 : (so.scan ? 3 : 2) * so.passes;
        const uint64_t share = (bytes / launches + kClearStep) / kClearStep * kClearStep;
        uint64_t cleared = 0;
        SortPass p = {};
        // blocks of the next launch: `work` of them for the sort
        const auto with_clear = [&](uint32_t work) {
            const uint64_t end = cleared + share < bytes ? cleared + share : bytes;
            const uint64_t size = end - cleared;
            const uint64_t each = (size / kClearBlocks + kClearStep) / kClearStep * kClearStep;
            p.blocks = work;
            p.clear = {static_cast<char *>(table_grad), cleared, end, each};
            cleared = end;
            return dim3((unsigned)(work + (size + each - 1) / each));
        };
        p.ids = cells;
        p.id_type = id_type;
        p.num_cells = cells_n;
        p.counts = reinterpret_cast<uint32_t *>(at + lay.counts);
        p.totals = reinterpret_cast<uint32_t *>(at + lay.totals);
        p.n = n;
        p.tiles = so.tiles;
        p.bits = so.bits;
        p.passes = so.passes;
        p.scanned = so.scan;
        const auto pass = [&](uint32_t k) {
            p.shift = k * so.bits;
            p.out = reinterpret_cast<uint2 *>(at + lay.order[k & 1]);
            p.weight = k == 0 ? weight : p.weight_out;
            p.scale = k == 0 ? scale : 1.0f;
            if (weight) p.weight_out = reinterpret_cast<float *>(at + lay.factor[k & 1]);
        };
        if (alone) {
            pass(0);
            const dim3 grid = with_clear(n > 0 ? 1 : 0);
            if (n <= kTile)
                hipLaunchKernelGGL(sort_block_kernel<kSteps>, grid, dim3(kSortThreads),
                                   order_bytes(so.bits, 8 * kTile), s, p);
            else
                hipLaunchKernelGGL(sort_block_kernel<16>, grid, dim3(kSortThreads),
                                   order_bytes(so.bits, 8 * kOneBlock), s, p);
        } else {
            for (uint32_t k = 0; k < so.passes; ++k) {
                pass(k);
                dim3 grid = with_clear(so.tiles);
                hipLaunchKernelGGL(sort_count_kernel, grid, dim3(kSortThreads), 4u << so.bits, s, p);
                if (so.scan) {
                    grid = with_clear(((1u << so.bits) + 63u) / 64u);
                    hipLaunchKernelGGL(sort_scan_kernel, grid, dim3(64 * kScanParts), 0, s, p);
                }
                grid = with_clear(so.tiles);
                hipLaunchKernelGGL(sort_scatter_kernel, grid, dim3(kSortThreads),
                                   order_bytes(so.bits, 12 * kTile), s, p);
                p.ids = nullptr;
                p.in = p.out;
            }
            a.factor = p.weight_out;
        }
        a.weight = weight;
        a.order = p.out;
    }
    with_piece(type, width, [&](auto t, auto kp) {
        using T = decltype(t);
        constexpr int kP = decltype(kp)::v;
        if (sum && n > 0)
            with_lanes(pieces, [&](auto lanes) {
                constexpr int kLanes = decltype(lanes)::v;
                a.grad = rows_grad;
                a.stride = rows_grad_stride;
                a.width = width;
                a.num_cells = cells_n;
                a.n = n;
                a.tile = tile_of(count, pieces);
                a.tiles = (n + a.tile - 1) / a.tile;
                a.scale = scale;
                a.partial = reinterpret_cast<float *>(at + lay.partial);
                a.table_grad = table_grad;
                a.table = table;
                a.table_stride = table_stride;
                a.weight_grad = beside ? weight_grad : nullptr;
                const dim3 grid((unsigned)(((uint64_t)a.tiles * kLanes + 255) / 256),
                                (pieces + kLanes - 1) / kLanes);
                hipLaunchKernelGGL((sums_kernel<T, kP, kLanes>), grid, dim3(256), 0, s, a);
                if (a.tiles > 1)
                    hipLaunchKernelGGL((join_rows_kernel<T, kP, kLanes>), grid, dim3(256), 0, s, a);
            });
        if (weight_grad && n > 0 && !beside) {
            // rows of no elements: as if no id named a cell
            RowsArgs w = {table, table_stride, width ? cells_n : 0u, width,
                          divisor(width ? pieces : 1u), cells, id_type, 0, count, 1, nullptr, scale,
                          nullptr};
            with_lanes(pieces, [&](auto lanes) {
                constexpr int kLanes = decltype(lanes)::v;
                constexpr uint64_t kIds = 256 / kLanes * kUnroll; // of a block
                for (uint64_t r = 0; r < count; r += kIds * kWindow) {
                    w.first = r;
                    w.count = count - r < kIds * kWindow ? count - r : kIds * kWindow;
                    hipLaunchKernelGGL((weight_grad_kernel<T, kP, kLanes>),
                                       dim3((unsigned)((w.count + kIds - 1) / kIds)), dim3(256), 0,
                                       s, w, static_cast<const T *>(rows_grad), rows_grad_stride,
                                       weight_grad);
                }
            });
        }
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "cell_rows_backward");
}

} // extern "C"
