// Rows in the order of the experts that they go to, and back.
//
// Entry e = K i + k is the k-th choice of row i; its group is the expert's id.  Entries
// in order (by group, those of one group as they came, those of none last):
//
//   place[e]   where entry e stands; -1 - place where it names no group
//   offset[g]  how many entries stand before group g's (offset[G]: that name a group)
//   rows:      y[place[K i + k], :] = x[i, :]                  (0 for an entry of none)
//   combine:   out[i, :] = sum_k w[i, k] y[place[K i + k], :]  (entries of none left out)
//   backward:  y_grad[place[K i + k], :] = w[i, k] out_grad[i, :]
//              w_grad[i, k] = <out_grad[i, :], y[place[K i + k], :]>
//
// The order comes from counting, not from atomics that return a place: every run gives
// the same.  Sums are fp32, over k in order, rounded to the rows' type once.
#include "head_device.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;
using namespace sdfoam_hip::head;

namespace {

// ---- the order --------------------------------------------------------------------

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t kSteps = 4;                  // entries a thread
constexpr uint32_t kTile = kSteps * kThreads;   // entries a block
// Up to so many tiles, each tile's block adds up the counts of all of them itself,
// which saves the scan's launch.  Microseconds with its own sums and with the scan: 65,536
// entries of 64 groups 10 and 12, of 2,048 groups 14 and 15; 262,144 entries (64 tiles) 12 and
// 14, 20 and 17; 524,288 the same and 28 and 18.
constexpr uint32_t kFewTiles = 64;
constexpr uint32_t kScanParts = 16;

struct OrderArgs {
    const void *ids;
    int id_type;
    uint32_t n, groups, tiles;
    uint32_t *counts; // [tiles][groups + 1]; the last: entries of no group
    uint32_t *totals; // [groups + 1]; NULL: counts as they were made
    int32_t *places;  // NULL: not wanted
    int32_t *entries; // by place; NULL: not wanted
    int32_t *group_of; // by place, -1 for none; NULL: not wanted
    int32_t *offsets;
};

__device__ __forceinline__ uint32_t key_of(const OrderArgs &a, uint32_t i) {
    const int32_t g = load_id(a.ids, a.id_type, i, a.groups);
    return g < 0 ? a.groups : (uint32_t)g;
}

__global__ __launch_bounds__(kThreads) void order_count_kernel(OrderArgs a) {
    extern __shared__ uint32_t hist[];
    const uint32_t keys = a.groups + 1;
    for (uint32_t g = threadIdx.x; g < keys; g += kThreads) hist[g] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t i = blockIdx.x * kTile + s * kThreads + threadIdx.x;
        if (i < a.n) atomicAdd(&hist[key_of(a, i)], 1u);
    }
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < keys; g += kThreads)
        a.counts[(uint64_t)blockIdx.x * keys + g] = hist[g];
}

// Per group, the exclusive sums over the tiles and the total: 64 groups a block,
// kScanParts threads each with a run of tiles.
__global__ __launch_bounds__(64 * kScanParts) void order_scan_kernel(OrderArgs a) {
    __shared__ uint32_t sums[kScanParts][64];
    const uint32_t keys = a.groups + 1;
    const uint32_t g = blockIdx.x * 64u + (threadIdx.x & 63u), part = threadIdx.x >> 6;
    const uint32_t each = (a.tiles + kScanParts - 1) / kScanParts;
    const uint32_t lo = min(part * each, a.tiles), hi = min(lo + each, a.tiles);
    uint32_t s = 0;
    if (g < keys)
#pragma unroll 8
        for (uint32_t t = lo; t < hi; ++t) s += a.counts[(uint64_t)t * keys + g];
    sums[part][threadIdx.x & 63u] = s;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (uint32_t k = 0; k < kScanParts; ++k) {
        const uint32_t v = sums[k][threadIdx.x & 63u];
        if (k < part) before += v;
        total += v;
    }
    if (g >= keys) return;
    if (part == 0) a.totals[g] = total;
#pragma unroll 8
    for (uint32_t t = lo; t < hi; ++t) {
        const uint32_t v = a.counts[(uint64_t)t * keys + g];
        a.counts[(uint64_t)t * keys + g] = before;
        before += v;
    }
}

// LDS: [keys] where the tile's entries of a group begin, [keys] totals and their sums,
// [kWaves][keys] 16-bit counts of the waves.
inline size_t place_lds(uint32_t groups) {
    const size_t keys = groups + 1;
    return keys * 8 + 64 * 4 + (kWaves * keys * 2 + 3) / 4 * 4;
}

// The places of one tile's entries.  A wave has 256 neighbouring entries, 64 a step;
// lanes with the same group find each other by ballots of the group's bits, and count
// on from the wave's entries before.  A wave holds at most 256 of a group: 16 bits.
__global__ __launch_bounds__(kThreads) void order_place_kernel(OrderArgs a) {
    extern __shared__ uint32_t lds[];
    const uint32_t keys = a.groups + 1;
    uint32_t *first = lds, *total = lds + keys, *parts = total + keys;
    uint16_t *count = reinterpret_cast<uint16_t *>(parts + 64);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t k = threadIdx.x; k < (kWaves * keys + 1) / 2; k += kThreads)
        reinterpret_cast<uint32_t *>(count)[k] = 0;
    uint32_t key[kSteps], rank[kSteps];
    const uint32_t base = blockIdx.x * kTile + wave * (64 * kSteps);
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t i = base + s * 64 + lane;
        key[s] = i < a.n ? key_of(a, i) : ~0u;
    }
    __syncthreads();
    uint16_t *mine = count + wave * keys;
    const uint32_t bits = 32 - __clz(a.groups);
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
        uint64_t peers = __ballot(key[s] != ~0u);
        for (uint32_t b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(key[s] >> b & 1u);
            peers &= key[s] >> b & 1u ? set : ~set;
        }
        const uint32_t below = __popcll(peers & ((1ull << lane) - 1));
        if (key[s] != ~0u) {
            const uint32_t before = mine[key[s]];
            rank[s] = before + below;
        }
        wave_sync();
        if (key[s] != ~0u && below == 0)
            mine[key[s]] = (uint16_t)(rank[s] + __popcll(peers));
        wave_sync();
    }
    __syncthreads();
    // by group: the waves' counts become sums of those before, the tiles' as well
    for (uint32_t g = threadIdx.x; g < keys; g += kThreads) {
        uint32_t own = 0;
        for (uint32_t w = 0; w < kWaves; ++w) {
            const uint32_t c = count[w * keys + g];
            count[w * keys + g] = (uint16_t)own;
            own += c;
        }
        uint32_t before = 0, all = own;
        if (a.totals) {
            before = a.counts[(uint64_t)blockIdx.x * keys + g];
            all = a.totals[g];
        } else if (a.tiles > 1) {
            all = 0;
#pragma unroll 8
            for (uint32_t t = 0; t < a.tiles; ++t) {
                const uint32_t c = a.counts[(uint64_t)t * keys + g];
                if (t < blockIdx.x) before += c;
                all += c;
            }
        }
        first[g] = before;
        total[g] = all;
    }
    __syncthreads();
    // where each group begins: exclusive sums of the totals, a run of groups a thread
    const uint32_t each = (keys + kThreads - 1) / kThreads;
    const uint32_t lo = min(threadIdx.x * each, keys), hi = min(lo + each, keys);
    uint32_t sum = 0;
    for (uint32_t g = lo; g < hi; ++g) sum += total[g];
    uint32_t run = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t v = __shfl_up(run, d);
        if ((int)lane >= d) run += v;
    }
    if (lane == 63) parts[wave] = run;
    __syncthreads();
    run -= sum;
    for (uint32_t w = 0; w < wave; ++w) run += parts[w];
    for (uint32_t g = lo; g < hi; ++g) {
        if (blockIdx.x == 0) a.offsets[g] = (int32_t)run;
        first[g] += run;
        run += total[g];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
        if (key[s] == ~0u) continue;
        const uint32_t i = base + s * 64 + lane;
        const int32_t p = (int32_t)(first[key[s]] + mine[key[s]] + rank[s]);
        const bool named = key[s] < a.groups;
        if (a.places) a.places[i] = named ? p : -1 - p;
        if (a.entries) a.entries[p] = (int32_t)i;
        if (a.group_of) a.group_of[p] = named ? (int32_t)key[s] : -1;
    }
}

uint32_t order_tiles(uint64_t n) { return (uint32_t)((n + kTile - 1) / kTile); }

__global__ __launch_bounds__(256) void order_none_kernel(int32_t *offsets, uint32_t keys) {
    const uint32_t g = blockIdx.x * 256 + threadIdx.x;
    if (g < keys) offsets[g] = 0;
}

} // namespace

namespace sdfoam_hip {
namespace head {

size_t order_scratch_bytes(uint64_t n, uint32_t groups) {
    const uint32_t tiles = order_tiles(n);
    if (tiles <= 1) return 0;
    return round_up(((size_t)tiles + 1) * (groups + 1) * 4);
}

hipError_t launch_order(int id_type, const void *ids, uint64_t n, uint32_t groups,
                        int32_t *places, int32_t *entries, int32_t *group_of, int32_t *offsets,
                        void *scratch, hipStream_t s) {
    const uint32_t keys = groups + 1;
    if (n == 0) {
        order_none_kernel<<<(keys + 255) / 256, 256, 0, s>>>(offsets, keys);
        return hipGetLastError();
    }
    OrderArgs a = {};
    a.ids = ids;
    a.id_type = id_type;
    a.n = (uint32_t)n;
    a.groups = groups;
    a.tiles = order_tiles(n);
    a.places = places;
    a.entries = entries;
    a.group_of = group_of;
    a.offsets = offsets;
    if (a.tiles > 1) {
        a.counts = static_cast<uint32_t *>(scratch);
        order_count_kernel<<<a.tiles, kThreads, keys * 4, s>>>(a);
        if (a.tiles > kFewTiles) {
            a.totals = a.counts + (uint64_t)a.tiles * keys;
            order_scan_kernel<<<(keys + 63) / 64, 64 * kScanParts, 0, s>>>(a);
        }
    }
    const size_t lds = place_lds(groups);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(
            reinterpret_cast<const void *>(order_place_kernel),
            hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    order_place_kernel<<<a.tiles, kThreads, lds, s>>>(a);
    return hipGetLastError();
}

} // namespace head
} // namespace sdfoam_hip

namespace {

// ---- rows and back ------------------------------------------------------------------

struct RowArgs {
    const void *in;   // rows: x; combine: y; backward: out_grad
    uint64_t stride;  // of `in`
    const void *sorted; // backward: y; NULL: no weight_grad
    uint64_t sorted_stride;
    const int32_t *places;
    const float *weight; // NULL: 1
    void *out;
    float *weight_grad;
    uint64_t rows, entries;
    uint32_t choices, width;
    uint32_t lanes; // of a row (a power of two, at most 64)
};

// 16 bytes of a row, or one element of a row shorter than that.  A last piece that would
// pass the row's end ends there.
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
// Rows that fill the caches go past them.  131,072 rows of 1,024 bf16 written from 16,384:
// 89 -> 54 us.
constexpr uint64_t kPastBytes = 128ull << 20;
template <bool kPast, typename T, int kP>
__device__ __forceinline__ void store_piece_if(T *p, const Piece<T, kP> &c) {
    if constexpr (kPast && sizeof(c) == 16) store_past<sizeof(T)>(p, c);
    else store_piece<T, kP>(p, c);
}

// A group of `lanes` per row; a lane has every lanes-th piece of it.
#define ROW_OF_GROUP                                                                       \
    const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / a.lanes;               \
    const uint32_t lane = threadIdx.x % a.lanes;                                           \
    const uint32_t pieces = (a.width + kP - 1) / kP

template <typename T, int kP, bool kPast> __global__ __launch_bounds__(256) void spread_kernel(RowArgs a) {
    ROW_OF_GROUP;
    if (i >= a.rows) return;
    const T *x = static_cast<const T *>(a.in) + i * a.stride;
    for (uint32_t c = lane; c < pieces; c += a.lanes) {
        const uint32_t col = min(c * kP, a.width - kP);
        const Piece<T, kP> v = load_piece<T, kP>(x + col), zero = {};
        for (uint32_t k = 0; k < a.choices; ++k) {
            const int32_t p = a.places[i * a.choices + k];
            const uint64_t at = p < 0 ? -1 - (int64_t)p : p;
            if (at >= a.entries) continue; // no place of these rows
            store_piece_if<kPast, T, kP>(static_cast<T *>(a.out) + at * a.width + col, p < 0 ? zero : v);
        }
    }
}

template <typename T, int kP> __global__ __launch_bounds__(256) void combine_kernel(RowArgs a) {
    ROW_OF_GROUP;
    if (i >= a.rows) return;
    T *out = static_cast<T *>(a.out) + i * a.width;
    for (uint32_t c = lane; c < pieces; c += a.lanes) {
        const uint32_t col = min(c * kP, a.width - kP);
        float sum[kP] = {};
        for (uint32_t k = 0; k < a.choices; ++k) {
            const int32_t p = a.places[i * a.choices + k];
            if (p < 0 || (uint64_t)p >= a.entries) continue;
            const float w = a.weight ? a.weight[i * a.choices + k] : 1.0f;
            const Piece<T, kP> v =
                load_piece<T, kP>(static_cast<const T *>(a.in) + (uint64_t)p * a.stride + col);
#pragma unroll
            for (int e = 0; e < kP; ++e) sum[e] = fmaf(w, (float)v.v[e], sum[e]);
        }
        Piece<T, kP> o;
#pragma unroll
        for (int e = 0; e < kP; ++e) o.v[e] = (T)sum[e];
        store_piece<T, kP>(out + col, o);
    }
}

template <typename T, int kP, bool kPast>
__global__ __launch_bounds__(256) void combine_backward_kernel(RowArgs a) {
    ROW_OF_GROUP;
    const bool in_range = i < a.rows;
    for (uint32_t k = 0; k < a.choices; ++k) {
        float dot = 0.0f;
        int32_t p = -1;
        if (in_range) {
            const T *g = static_cast<const T *>(a.in) + i * a.stride;
            p = a.places[i * a.choices + k];
            const uint64_t at = p < 0 ? -1 - (int64_t)p : p;
            const float w = a.weight ? a.weight[i * a.choices + k] : 1.0f;
            if (at < a.entries) {
                for (uint32_t c = lane; c < pieces; c += a.lanes) {
                    const uint32_t col = min(c * kP, a.width - kP);
                    const Piece<T, kP> v = load_piece<T, kP>(g + col);
                    if (a.out) {
                        Piece<T, kP> o;
#pragma unroll
                        for (int e = 0; e < kP; ++e)
                            o.v[e] = (T)(p < 0 ? 0.0f : w * (float)v.v[e]);
                        store_piece_if<kPast, T, kP>(static_cast<T *>(a.out) + at * a.width + col, o);
                    }
                    if (a.sorted && p >= 0) {
                        const Piece<T, kP> y = load_piece<T, kP>(
                            static_cast<const T *>(a.sorted) + at * a.sorted_stride + col);
#pragma unroll
                        for (int e = 0; e < kP; ++e) // not those of the piece before
                            if (col + e >= c * kP) dot = fmaf((float)v.v[e], (float)y.v[e], dot);
                    }
                }
            }
        }
        if (a.sorted) {
            for (uint32_t d = a.lanes >> 1; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
            if (in_range && lane == 0) a.weight_grad[i * a.choices + k] = p < 0 ? 0.0f : dot;
        }
    }
}

template <typename F> hipError_t with_pieces(int type, RowArgs &a, hipStream_t s, F launch) {
    return with_type(type, [&](auto t) {
        typedef decltype(t) T;
        constexpr uint32_t kP = 16 / sizeof(T);
        const bool whole = a.width >= kP;
        const uint32_t pieces = whole ? (a.width + kP - 1) / kP : a.width;
        a.lanes = 1;
        while (a.lanes < 64 && a.lanes < pieces) a.lanes *= 2;
        const uint64_t rows_block = 256 / a.lanes;
        const uint64_t blocks = (a.rows + rows_block - 1) / rows_block;
        // a launch holds fewer than 2^32 threads
        constexpr uint64_t kWindow = 1ull << 23;
        RowArgs b = a;
        for (uint64_t first = 0; first < blocks; first += kWindow) {
            const uint64_t i = first * rows_block;
            const uint64_t now = blocks - first < kWindow ? blocks - first : kWindow;
            b.rows = a.rows - i < now * rows_block ? a.rows - i : now * rows_block;
            b.places = a.places + i * a.choices;
            if (a.weight) b.weight = a.weight + i * a.choices;
            if (a.weight_grad) b.weight_grad = a.weight_grad + i * a.choices;
            launch(t, b, i, (uint32_t)now, whole);
        }
        return hipGetLastError();
    });
}

int check_rows(const char *call, int type, uint64_t rows, uint32_t choices, uint32_t width) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: type must be SDF_TYPE_*", call);
    if (width > 1u << 18) return fail(SDF_E_INVALID, "%s takes rows of at most 2^18 elements", call);
    if (rows >= 1ull << 31 || rows * choices >= 1ull << 31)
        return fail(SDF_E_INVALID, "%s takes fewer than 2^31 entries", call);
    return SDF_OK;
}

} // namespace

extern "C" {

size_t sdf_expert_order_scratch_bytes(uint64_t count, uint32_t num_experts) {
    if (count >= 1ull << 31 || num_experts > SDF_MAX_EXPERTS) return 0;
    return order_scratch_bytes(count, num_experts);
}

int sdf_expert_order(int id_type, const void *experts, uint64_t count, uint32_t num_experts,
                     int32_t *places, int32_t *offsets, void *scratch, size_t scratch_bytes,
                     void *stream) {
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "id_type must be SDF_ID_*");
    if (num_experts > SDF_MAX_EXPERTS)
        return fail(SDF_E_INVALID, "at most %u experts (got %u)", SDF_MAX_EXPERTS, num_experts);
    if (count >= 1ull << 31)
        return fail(SDF_E_INVALID, "sdf_expert_order takes fewer than 2^31 entries");
    if (!offsets || (count > 0 && (!experts || !places)))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const int rc = check_scratch(scratch, scratch_bytes, order_scratch_bytes(count, num_experts));
    if (rc != SDF_OK) return rc;
    const hipError_t e = launch_order(id_type, experts, count, num_experts, places, nullptr,
                                      nullptr, offsets, scratch, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? SDF_OK : hip_fail(e, "expert_order");
}

int sdf_expert_rows(int type, const void *rows, uint64_t rows_stride, uint64_t count,
                    uint32_t choices, uint32_t width, const int32_t *places, void *sorted,
                    void *stream) {
    const int rc = check_rows("sdf_expert_rows", type, count, choices, width);
    if (rc != SDF_OK) return rc;
    if (count == 0 || choices == 0 || width == 0) return SDF_OK;
    if (!rows || !places || !sorted) return fail(SDF_E_INVALID, "NULL pointer argument");
    RowArgs a = {};
    a.in = rows;
    a.stride = rows_stride;
    a.places = places;
    a.out = sorted;
    a.rows = count;
    a.entries = count * choices;
    a.choices = choices;
    a.width = width;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e =
        with_pieces(type, a, s, [&](auto t, RowArgs &b, uint64_t i, uint32_t blocks, bool whole) {
            typedef decltype(t) T;
            b.in = static_cast<const T *>(a.in) + i * a.stride;
            const bool past = a.entries * a.width * sizeof(T) >= kPastBytes;
            if (whole && past) spread_kernel<T, 16 / sizeof(T), true><<<blocks, 256, 0, s>>>(b);
            else if (whole) spread_kernel<T, 16 / sizeof(T), false><<<blocks, 256, 0, s>>>(b);
            else spread_kernel<T, 1, false><<<blocks, 256, 0, s>>>(b);
        });
    return e == hipSuccess ? SDF_OK : hip_fail(e, "expert_rows");
}

int sdf_expert_combine(int type, const void *sorted, uint64_t sorted_stride, uint64_t count,
                       uint32_t choices, uint32_t width, const int32_t *places,
                       const float *weight, void *out, void *stream) {
    const int rc = check_rows("sdf_expert_combine", type, count, choices, width);
    if (rc != SDF_OK) return rc;
    if (count == 0 || width == 0) return SDF_OK;
    if (!out || (choices > 0 && (!sorted || !places)))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    RowArgs a = {};
    a.in = sorted;
    a.stride = sorted_stride;
    a.places = places;
    a.weight = weight;
    a.out = out;
    a.rows = count;
    a.entries = count * choices;
    a.choices = choices;
    a.width = width;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e =
        with_pieces(type, a, s, [&](auto t, RowArgs &b, uint64_t i, uint32_t blocks, bool whole) {
            typedef decltype(t) T;
            b.out = static_cast<T *>(a.out) + i * a.width;
            if (whole) combine_kernel<T, 16 / sizeof(T)><<<blocks, 256, 0, s>>>(b);
            else combine_kernel<T, 1><<<blocks, 256, 0, s>>>(b);
        });
    return e == hipSuccess ? SDF_OK : hip_fail(e, "expert_combine");
}

int sdf_expert_combine_backward(int type, const void *out_grad, uint64_t out_grad_stride,
                                const void *sorted, uint64_t sorted_stride, uint64_t count,
                                uint32_t choices, uint32_t width, const int32_t *places,
                                const float *weight, void *sorted_grad, float *weight_grad,
                                void *stream) {
    const int rc = check_rows("sdf_expert_combine_backward", type, count, choices, width);
    if (rc != SDF_OK) return rc;
    if (count == 0 || choices == 0 || (!sorted_grad && !weight_grad)) return SDF_OK;
    if (!places || (width > 0 && (!out_grad || (weight_grad && !sorted))))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    RowArgs a = {};
    a.in = out_grad;
    a.stride = out_grad_stride;
    // rows of no elements: the weights' gradients are 0, nothing is read
    a.sorted = weight_grad ? (width > 0 ? sorted : places) : nullptr;
    a.sorted_stride = sorted_stride;
    a.places = places;
    a.weight = weight;
    a.out = sorted_grad;
    a.weight_grad = weight_grad;
    a.rows = count;
    a.entries = count * choices;
    a.choices = choices;
    a.width = width;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e =
        with_pieces(type, a, s, [&](auto t, RowArgs &b, uint64_t i, uint32_t blocks, bool whole) {
            typedef decltype(t) T;
            b.in = static_cast<const T *>(a.in) + i * a.stride;
            const bool past = a.entries * a.width * sizeof(T) >= kPastBytes;
            if (whole && past) combine_backward_kernel<T, 16 / sizeof(T), true><<<blocks, 256, 0, s>>>(b);
            else if (whole) combine_backward_kernel<T, 16 / sizeof(T), false><<<blocks, 256, 0, s>>>(b);
            else combine_backward_kernel<T, 1, false><<<blocks, 256, 0, s>>>(b);
        });
    return e == hipSuccess ? SDF_OK : hip_fail(e, "expert_combine_backward");
}

} // extern "C"
