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
constexpr uint64_t kWindow = 1ull << 22; // blocks a launch: it holds fewer than 2^32 threads
constexpr uint32_t kMaxWidth = 1u << 18; // of a row: Divisor's range

// One lane per piece of a row, kUnroll of them in flight: bound by the bytes of
// the rows read and written (the ids come once per row, from L1 after that).
template <typename T, int kP> __global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
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
            store_piece<T, kP>(out + (r0 + row[u]) * a.width + col[u], o);
        }
    }
}

// ---- the sort of the ids: stable, least significant digit first ---------------

constexpr uint32_t kTile = 4096;     // keys of one block
constexpr uint32_t kMaxBits = 11;    // of a digit
constexpr uint32_t kScanTiles = 16;  // threads that share a digit's tiles

struct SortPass {
    const void *ids; // first pass: the caller's ids; NULL: keys_in, index_in
    int id_type;
    uint32_t num_cells;
    const uint32_t *keys_in, *index_in;
    uint32_t *keys_out, *index_out;
    uint32_t *counts; // [tiles][digits], after the scan those of the tiles before
    uint32_t *totals; // [digits]
    uint8_t *named;   // [num_cells] whether an id names the cell: cleared in the
                      // first pass, written in the last
    uint32_t n, tiles, shift, bits;
    bool clear, mark;
};

// no cell sorts last
__device__ __forceinline__ uint32_t sort_key(const SortPass &p, uint32_t i) {
    if (!p.ids) return p.keys_in[i];
    const int32_t c = load_id(p.ids, p.id_type, i, p.num_cells);
    return c < 0 ? p.num_cells : (uint32_t)c;
}

__global__ __launch_bounds__(256) void sort_count_kernel(SortPass p) {
    __shared__ uint32_t hist[1u << kMaxBits];
    const uint32_t digits = 1u << p.bits;
    for (uint32_t d = threadIdx.x; d < digits; d += 256u) hist[d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile;
#pragma unroll 4
    for (uint32_t j = threadIdx.x; j < kTile; j += 256u)
        if (base + j < p.n)
            atomicAdd(&hist[(sort_key(p, base + j) >> p.shift) & (digits - 1)], 1u);
    if (p.clear) { // 16 bytes a thread; the array is padded to them
        uint4 *named = reinterpret_cast<uint4 *>(p.named);
        const uint32_t words = (p.num_cells + 15u) / 16u;
        for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < words; i += gridDim.x * 256u)
            named[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += 256u)
        p.counts[(uint64_t)blockIdx.x * digits + d] = hist[d];
}

// Per digit, the exclusive sums over the tiles and the total: 64 digits a
// block, kScanTiles threads each with a run of tiles.
__global__ __launch_bounds__(64 * kScanTiles) void sort_scan_kernel(SortPass p) {
    __shared__ uint32_t sums[kScanTiles][64];
    const uint32_t digits = 1u << p.bits;
    const uint32_t d = blockIdx.x * 64u + (threadIdx.x & 63u), part = threadIdx.x >> 6;
    const uint32_t each = (p.tiles + kScanTiles - 1) / kScanTiles;
    const uint32_t lo = min(part * each, p.tiles), hi = min(lo + each, p.tiles);
    uint32_t s = 0;
    if (d < digits)
#pragma unroll 8
        for (uint32_t t = lo; t < hi; ++t) s += p.counts[(uint64_t)t * digits + d];
    sums[part][threadIdx.x & 63u] = s;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (uint32_t k = 0; k < kScanTiles; ++k) {
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

// Each wavefront ranks 1,024 consecutive keys: the lanes of equal digits find
// each other by one ballot per bit, a counter per digit in LDS carries the
// rank from one step of 64 keys to the next.
__global__ __launch_bounds__(256) void sort_scatter_kernel(SortPass p) {
    __shared__ uint32_t seen[4][1u << kMaxBits];
    __shared__ uint32_t waves[4];
    const uint32_t digits = 1u << p.bits;
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    for (uint32_t d = threadIdx.x; d < digits; d += 256u)
        for (uint32_t k = 0; k < 4u; ++k) seen[k][d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile + w * (kTile / 4);
    uint32_t key[16], rank[16];
#pragma unroll
    for (uint32_t r = 0; r < 16u; ++r) {
        const uint32_t i = base + r * 64u + lane;
        key[r] = i < p.n ? sort_key(p, i) : 0u;
    }
#pragma unroll
    for (uint32_t r = 0; r < 16u; ++r) {
        const bool in = base + r * 64u + lane < p.n;
        const uint32_t d = (key[r] >> p.shift) & (digits - 1);
        uint64_t same = __ballot(in);
        for (uint32_t b = 0; b < p.bits; ++b) {
            const uint64_t set = __ballot((d >> b) & 1u);
            same &= (d >> b) & 1u ? set : ~set;
        }
        const uint32_t below = __popcll(same & ((1ull << lane) - 1ull));
        uint32_t first = 0;
        if (in && below == 0) first = atomicAdd(&seen[w][d], (uint32_t)__popcll(same));
        const int leader = in ? __ffsll((unsigned long long)same) - 1 : (int)lane;
        rank[r] = __shfl(first, leader) + below;
        if (p.mark) { // ids of one cell stand side by side by now
            const uint32_t left = __shfl_up(key[r], 1);
            if (in && key[r] < p.num_cells && (lane == 0 || left != key[r])) p.named[key[r]] = 1;
        }
    }
    __syncthreads();
    // where each digit starts: runs of digits / 256 of them per thread
    const uint32_t each = (digits + 255u) / 256u, lo = threadIdx.x * each;
    uint32_t mine = 0;
    for (uint32_t d = lo; d < lo + each && d < digits; ++d) mine += p.totals[d];
    uint32_t s = mine;
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63u) waves[w] = s;
    __syncthreads();
    uint32_t start = s - mine;
    for (uint32_t k = 0; k < w; ++k) start += waves[k];
    for (uint32_t d = lo; d < lo + each && d < digits; ++d) {
        uint32_t at = start + p.counts[(uint64_t)blockIdx.x * digits + d];
        for (uint32_t k = 0; k < 4u; ++k) {
            const uint32_t c = seen[k][d];
            seen[k][d] = at;
            at += c;
        }
        start += p.totals[d];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < 16u; ++r) {
        const uint32_t i = base + r * 64u + lane;
        if (i >= p.n) continue;
        const uint32_t to = seen[w][(key[r] >> p.shift) & (digits - 1)] + rank[r];
        p.keys_out[to] = key[r];
        p.index_out[to] = p.ids ? i : p.index_in[i];
    }
}

// ---- the sums -------------------------------------------------------------------

// The sorted ids in tiles of `tile` positions, a tile to kLanes lanes (which
// hold a row, or 64 pieces of it).  A cell whose positions all lie in one tile
// is summed and written there.  Of a cell that goes on in other tiles, each
// tile keeps its sum in fp32: slot 0 where the cell began in an earlier tile,
// slot 1 where it begins here; join_rows_kernel adds them.
struct SumsArgs {
    const void *grad;
    uint64_t stride;
    uint32_t width, num_cells;
    const uint32_t *keys, *index; // padded to whole tiles, the padding not read as ids
    uint32_t n, tile, tiles;
    const float *weight;
    float scale;
    float *partial; // [tiles][2][width]
    void *table_grad;
    const void *table; // with weight_grad
    uint64_t table_stride;
    float *weight_grad; // NULL: not formed here
    const uint8_t *named;
    uint32_t sum_blocks; // the blocks after them clear the cells that no id names
    uint32_t clear_rows; // rows a block
    Divisor pieces;
};

constexpr int kBatch = 8; // rows in flight per lane

template <typename T, int kP, int kLanes>
__device__ __forceinline__ void sum_tile(const SumsArgs &a, uint32_t tile, uint32_t piece, uint32_t l) {
    const T *grad = static_cast<const T *>(a.grad);
    T *out = static_cast<T *>(a.table_grad);
    const bool mine = piece * kP < a.width; // lanes past the row hold nothing
    const uint32_t col = mine ? column<kP>(piece, a.width) : 0u;
    const uint32_t p0 = tile * a.tile, p1 = min(p0 + a.tile, a.n);
    const uint32_t before = p0 > 0 ? a.keys[p0 - 1] : a.num_cells;
    const uint32_t after = p1 < a.n ? a.keys[p1] : a.num_cells;
    float acc[kP] = {};
    uint32_t cell = a.keys[p0];
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
            const uint32_t at = min(p + b, p1 - 1);
            key[b] = a.keys[at];
            index[b] = a.index[at];
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const bool live = p + b < p1 && key[b] < a.num_cells;
            f[b] = live ? (a.weight ? a.scale * a.weight[index[b]] : a.scale) : 0.0f;
            g[b] = {};
            if (live && mine) g[b] = load_piece<T, kP>(grad + (uint64_t)index[b] * a.stride + col);
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
                if (l == b % kLanes && p + b < p1) a.weight_grad[index[b]] = a.scale * s;
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
    if (blockIdx.x < a.sum_blocks) {
        const uint32_t tile = (blockIdx.x * 256u + threadIdx.x) / kLanes, l = threadIdx.x % kLanes;
        if (tile < a.tiles) sum_tile<T, kP, kLanes>(a, tile, blockIdx.y * kLanes + l, l);
        return;
    }
    if (blockIdx.y > 0) return;
    const uint64_t r0 = (uint64_t)(blockIdx.x - a.sum_blocks) * a.clear_rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.clear_rows, a.num_cells - r0);
    const Piece<T, kP> zero = {};
    for (uint32_t t = threadIdx.x; t < rows * a.pieces.d; t += 256u) {
        const uint32_t row = t / a.pieces;
        if (a.n > 0 && a.named[r0 + row]) continue;
        store_piece<T, kP>(static_cast<T *>(a.table_grad) + (r0 + row) * a.width +
                               column<kP>(t - row * a.pieces.d, a.width),
                           zero);
    }
}

constexpr uint32_t kLong = 16; // tiles that one group adds by itself

// The cells that go on past the tile they begin in: their tiles' sums in order.
// A cell of more than kLong tiles is added by the whole block, every group a
// share of its tiles.
template <typename T, int kP, int kLanes>
__global__ __launch_bounds__(256) void join_rows_kernel(SumsArgs a) {
    constexpr uint32_t kGroups = 256 / kLanes;
    __shared__ uint32_t list[kGroups];
    __shared__ uint32_t listed;
    __shared__ float sums[kGroups][kLanes * kP];
    const uint32_t g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
    const uint32_t tile = blockIdx.x * kGroups + g, piece = blockIdx.y * kLanes + l;
    const bool mine = piece * kP < a.width;
    const uint32_t col = mine ? column<kP>(piece, a.width) : 0u;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const auto slot = [&](uint32_t t, uint32_t k) {
        return a.partial + ((uint64_t)t * 2 + k) * a.width + col;
    };
    const auto starts = [&](uint32_t t) { return a.keys[(uint64_t)t * a.tile]; };
    const auto write = [&](uint32_t cell, const float *s) {
        if (!mine) return;
        Piece<T, kP> o;
#pragma unroll
        for (int e = 0; e < kP; ++e) o.v[e] = (T)s[e];
        store_piece<T, kP>(static_cast<T *>(a.table_grad) + (uint64_t)cell * a.width + col, o);
    };
    if (tile + 1 < a.tiles) {
        const uint32_t p0 = tile * a.tile, cell = a.keys[p0 + a.tile - 1];
        const bool whole = p0 > 0 && a.keys[p0 - 1] == cell; // then the tile is all of that cell
        if (cell < a.num_cells && starts(tile + 1) == cell && !whole) {
            if (tile + kLong < a.tiles && starts(tile + kLong) == cell) {
                if (l == 0) list[atomicAdd(&listed, 1u)] = tile;
            } else {
                float s[kP];
#pragma unroll
                for (int e = 0; e < kP; ++e) s[e] = slot(tile, 1)[e];
                for (uint32_t t = tile + 1; t < a.tiles && starts(t) == cell; ++t) {
                    const float *x = slot(t, 0);
#pragma unroll
                    for (int e = 0; e < kP; ++e) s[e] += x[e];
                }
                write(cell, s);
            }
        }
    }
    __syncthreads();
    const uint32_t n = listed; // the order of the list does not matter: each has its own cell
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t first = list[i], cell = a.keys[(uint64_t)(first + 1) * a.tile - 1];
        uint32_t lo = first + kLong, hi = a.tiles; // the first tile that does not start with it
        while (lo + 1 < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (starts(mid) == cell) lo = mid;
            else hi = mid;
        }
        float s[kP] = {};
#pragma unroll 4
        for (uint32_t t = first + 1 + g; t < hi; t += kGroups) {
            const float *x = slot(t, 0);
#pragma unroll
            for (int e = 0; e < kP; ++e) s[e] += x[e];
        }
#pragma unroll
        for (int e = 0; e < kP; ++e) sums[g][l * kP + e] = s[e];
        __syncthreads();
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < kP; ++e) s[e] = slot(first, 1)[e];
            for (uint32_t k = 0; k < kGroups; ++k)
#pragma unroll
                for (int e = 0; e < kP; ++e) s[e] += sums[k][l * kP + e];
            write(cell, s);
        }
        __syncthreads();
    }
}

// The weights' gradient by itself, a wavefront per id: where the table's is not
// wanted, or a row is wider than a wavefront holds.
template <typename T, int kP>
__global__ __launch_bounds__(256) void weight_grad_kernel(RowsArgs a, const T *__restrict__ grad,
                                                          uint64_t grad_stride,
                                                          float *__restrict__ weight_grad) {
    const uint64_t i = a.first + (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    if (i >= a.first + a.count) return;
    const int32_t c = load_id(a.cells, a.id_type, i, a.num_cells);
    float s = 0.0f;
    if (c >= 0)
        for (uint32_t k = threadIdx.x & 63u; k < a.pieces.d; k += 64u) {
            const uint32_t col = column<kP>(k, a.width);
            const auto x = load_piece<T, kP>(grad + i * grad_stride + col);
            const auto y = load_piece<T, kP>(static_cast<const T *>(a.table) +
                                             (uint64_t)c * a.stride + col);
#pragma unroll
            for (int e = 0; e < kP; ++e)
                if (col + e >= k * kP) s = fmaf((float)x.v[e], (float)y.v[e], s);
        }
    s = group_sum<64>(s);
    if ((threadIdx.x & 63u) == 0) weight_grad[i] = a.scale * s;
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
};
Sort sort_of(uint64_t num_cells, uint64_t count) {
    uint32_t bits = 1; // of the largest key, num_cells
    while ((num_cells >> bits) != 0) ++bits;
    Sort s;
    s.passes = (bits + kMaxBits - 1) / kMaxBits;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.tiles = (uint32_t)((count + kTile - 1) / kTile);
    return s;
}

struct Layout {
    size_t keys[2], index[2], counts, totals, named, partial, bytes;
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
    for (int k = 0; k < 2; ++k) {
        o.keys[k] = take(4 * count);
        o.index[k] = take(4 * count);
    }
    o.counts = take(4ull * s.tiles << s.bits);
    o.totals = take(4ull << s.bits);
    o.named = take(num_cells);
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
    // 1,024 pieces a block, or 256 where that leaves CUs without one
    const uint64_t items = count * pieces < 1024 * 1024 ? 256 : 1024;
    a.per = (uint32_t)(items / pieces > 0 ? items / pieces : 1);
    with_piece(type, width, [&](auto t, auto p) {
        for (uint64_t r = 0; r < count; r += kWindow * a.per) {
            a.first = r;
            a.count = count - r < kWindow * a.per ? count - r : kWindow * a.per;
            hipLaunchKernelGGL((rows_kernel<decltype(t), decltype(p)::v>),
                               dim3((unsigned)((a.count + a.per - 1) / a.per)), dim3(256), 0,
                               static_cast<hipStream_t>(stream), a);
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
        (count > 0 && width > 0 && !rows_grad) || !scratch ||
        (weight_grad && num_cells > 0 && width > 0 && !table))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_cell_rows_backward_scratch_bytes(num_cells, width, count);
    if (scratch_bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    const size_t e_size = type_bytes(type);
    if (misaligned(rows_grad, e_size) || misaligned(table, e_size) || misaligned(table_grad, e_size))
        return fail(SDF_E_INVALID,
                    "cell_rows_backward: rows and tables must be aligned to their elements");
    if (misaligned(scratch, 256)) return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t n = (uint32_t)count, cells_n = (uint32_t)num_cells;
    const uint32_t pieces = pieces_of(type, width);
    const bool sum = table_grad && num_cells > 0 && width > 0;
    // the weights' gradient beside the sums, where a group of lanes sees whole rows
    const bool beside = sum && weight_grad && pieces <= 64;
    char *at = static_cast<char *>(scratch);
    const Layout lay = layout_of((int)type_bytes(type), num_cells, width, count);
    SumsArgs a = {};
    if (sum && n > 0) {
        const Sort so = sort_of(num_cells, count);
        SortPass p = {};
        p.ids = cells;
        p.id_type = id_type;
        p.num_cells = cells_n;
        p.counts = reinterpret_cast<uint32_t *>(at + lay.counts);
        p.totals = reinterpret_cast<uint32_t *>(at + lay.totals);
        p.named = reinterpret_cast<uint8_t *>(at + lay.named);
        p.n = n;
        p.tiles = so.tiles;
        p.bits = so.bits;
        for (uint32_t k = 0; k < so.passes; ++k) {
            p.shift = k * so.bits;
            p.clear = k == 0;
            p.mark = k + 1 == so.passes;
            p.keys_out = reinterpret_cast<uint32_t *>(at + lay.keys[k & 1]);
            p.index_out = reinterpret_cast<uint32_t *>(at + lay.index[k & 1]);
            hipLaunchKernelGGL(sort_count_kernel, dim3(so.tiles), dim3(256), 0, s, p);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(((1u << so.bits) + 63u) / 64u),
                               dim3(64 * kScanTiles), 0, s, p);
            hipLaunchKernelGGL(sort_scatter_kernel, dim3(so.tiles), dim3(256), 0, s, p);
            p.ids = nullptr;
            p.keys_in = p.keys_out;
            p.index_in = p.index_out;
        }
        a.keys = p.keys_out;
        a.index = p.index_out;
    }
    with_piece(type, width, [&](auto t, auto kp) {
        using T = decltype(t);
        constexpr int kP = decltype(kp)::v;
        if (sum)
            with_lanes(pieces, [&](auto lanes) {
                constexpr int kLanes = decltype(lanes)::v;
                a.grad = rows_grad;
                a.stride = rows_grad_stride;
                a.width = width;
                a.num_cells = cells_n;
                a.n = n;
                a.tile = tile_of(count, pieces);
                a.tiles = (n + a.tile - 1) / a.tile;
                a.weight = weight;
                a.scale = scale;
                a.partial = reinterpret_cast<float *>(at + lay.partial);
                a.table_grad = table_grad;
                a.table = table;
                a.table_stride = table_stride;
                a.weight_grad = beside ? weight_grad : nullptr;
                a.named = reinterpret_cast<const uint8_t *>(at + lay.named);
                a.pieces = divisor(pieces);
                a.sum_blocks = (uint32_t)(((uint64_t)a.tiles * kLanes + 255) / 256);
                a.clear_rows = pieces < 2048 ? 2048 / pieces : 1;
                const uint32_t clear = (cells_n + a.clear_rows - 1) / a.clear_rows;
                const uint32_t wide = (pieces + kLanes - 1) / kLanes;
                hipLaunchKernelGGL((sums_kernel<T, kP, kLanes>), dim3(a.sum_blocks + clear, wide),
                                   dim3(256), 0, s, a);
                if (a.tiles > 1)
                    hipLaunchKernelGGL((join_rows_kernel<T, kP, kLanes>), dim3(a.sum_blocks, wide),
                                       dim3(256), 0, s, a);
            });
        if (weight_grad && n > 0 && !beside) {
            // rows of no elements: as if no id named a cell
            RowsArgs w = {table, table_stride, width ? cells_n : 0u, width,
                          divisor(width ? pieces : 1u), cells, id_type, 0, count, 1, nullptr, scale,
                          nullptr};
            for (uint64_t r = 0; r < count; r += 4 * kWindow) {
                w.first = r;
                w.count = count - r < 4 * kWindow ? count - r : 4 * kWindow;
                hipLaunchKernelGGL((weight_grad_kernel<T, kP>), dim3((unsigned)((w.count + 3) / 4)),
                                   dim3(256), 0, s, w, static_cast<const T *>(rows_grad),
                                   rows_grad_stride, weight_grad);
            }
        }
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "cell_rows_backward");
}

} // extern "C"
