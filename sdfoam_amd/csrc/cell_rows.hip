// Rows of a per-cell table (features, embeddings) for a list of cells, and the
// gradients of the table and the weights.
//
//   rows[i, :]       = scale w_i table[c_i, :]          (0 where c_i is no cell)
//   table_grad[v, :] = sum over { i : c_i = v } of scale w_i rows_grad[i, :]
//   weight_grad[i]   = scale <table[c_i, :], rows_grad[i, :]>
//
// The table's gradient is formed cell by cell from the ids in sorted order
// (stable, so a cell's rows are added in the order of their positions): no
// atomics, the same bits on every run.  Sums are held in fp32 and rounded to
// the table's type once.
#include "label_device.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;

namespace {

constexpr uint32_t kTile = 4096; // keys of one block of the sort
constexpr uint32_t kDigits = 256;

template <typename T>
__global__ __launch_bounds__(256) void rows_kernel(const T *__restrict__ table, uint32_t num_cells,
                                                   uint32_t width, uint64_t stride,
                                                   const void *__restrict__ cells, int id_type,
                                                   uint64_t count, const float *__restrict__ weight,
                                                   float scale, T *__restrict__ rows) {
    const uint64_t t = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (t >= count * width) return;
    const uint64_t i = t / width;
    const uint32_t d = (uint32_t)(t - i * width);
    const int32_t c = load_id(cells, id_type, i, num_cells);
    if (c < 0) {
        rows[t] = (T)0.0f;
        return;
    }
    const float f = weight ? scale * weight[i] : scale;
    rows[t] = (T)(f * (float)table[(uint64_t)c * stride + d]);
}

// ---- the sort: least significant digit first, eight bits a pass -----------

struct SortPass {
    const void *ids; // first pass: the caller's ids; NULL: keys_in, index_in
    int id_type;
    uint32_t num_cells;
    const uint32_t *keys_in, *index_in;
    uint32_t *keys_out, *index_out;
    uint32_t *counts; // [kDigits][tiles], after the scan where each starts
    uint32_t n, tiles, shift;
};

// no cell sorts last
__device__ __forceinline__ uint32_t sort_key(const SortPass &p, uint32_t i) {
    if (!p.ids) return p.keys_in[i];
    const int32_t c = load_id(p.ids, p.id_type, i, p.num_cells);
    return c < 0 ? p.num_cells : (uint32_t)c;
}

__global__ __launch_bounds__(256) void sort_count_kernel(SortPass p) {
    __shared__ uint32_t hist[kDigits];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile;
    for (uint32_t j = threadIdx.x; j < kTile && base + j < p.n; j += 256u)
        atomicAdd(&hist[(sort_key(p, base + j) >> p.shift) & (kDigits - 1)], 1u);
    __syncthreads();
    p.counts[(uint64_t)threadIdx.x * p.tiles + blockIdx.x] = hist[threadIdx.x];
}

// Exclusive sums of counts, in place, by one block.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t *counts, uint32_t n) {
    __shared__ uint32_t waves[16];
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (uint32_t base = 0; base < n; base += 1024u) {
        const uint32_t i = base + threadIdx.x;
        const uint32_t v = i < n ? counts[i] : 0u;
        uint32_t s = v;
        for (uint32_t d = 1; d < 64u; d <<= 1) {
            const uint32_t o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        if (lane == 63u) waves[w] = s;
        __syncthreads();
        uint32_t before = carry, total = 0;
        for (uint32_t k = 0; k < 16u; ++k) {
            if (k < w) before += waves[k];
            total += waves[k];
        }
        if (i < n) counts[i] = before + s - v;
        carry += total;
        __syncthreads();
    }
}

// Each wavefront ranks 1,024 consecutive keys: the lanes of equal digits find
// each other by one ballot per bit, a counter per digit in LDS carries the
// rank from one step of 64 keys to the next.
__global__ __launch_bounds__(256) void sort_scatter_kernel(SortPass p) {
    __shared__ uint32_t seen[4][kDigits];
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    for (uint32_t k = 0; k < 4u; ++k) seen[k][threadIdx.x] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile + w * (kTile / 4);
    uint32_t key[16], rank[16];
    for (uint32_t r = 0; r < 16u; ++r) {
        const uint32_t i = base + r * 64u + lane;
        const bool in = i < p.n;
        key[r] = in ? sort_key(p, i) : 0u;
        const uint32_t d = (key[r] >> p.shift) & (kDigits - 1);
        uint64_t same = __ballot(in);
        for (uint32_t b = 0; b < 8u; ++b) {
            const uint64_t set = __ballot((d >> b) & 1u);
            same &= (d >> b) & 1u ? set : ~set;
        }
        const uint32_t below = __popcll(same & ((1ull << lane) - 1ull));
        uint32_t first = 0;
        if (in && below == 0) first = atomicAdd(&seen[w][d], (uint32_t)__popcll(same));
        const int leader = in ? __ffsll((unsigned long long)same) - 1 : (int)lane;
        rank[r] = __shfl(first, leader) + below;
    }
    __syncthreads();
    uint32_t at = p.counts[(uint64_t)threadIdx.x * p.tiles + blockIdx.x];
    for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t c = seen[k][threadIdx.x];
        seen[k][threadIdx.x] = at;
        at += c;
    }
    __syncthreads();
    for (uint32_t r = 0; r < 16u; ++r) {
        const uint32_t i = base + r * 64u + lane;
        if (i >= p.n) continue;
        const uint32_t to = seen[w][(key[r] >> p.shift) & (kDigits - 1)] + rank[r];
        p.keys_out[to] = key[r];
        p.index_out[to] = p.ids ? i : p.index_in[i];
    }
}

// ---- the sums --------------------------------------------------------------

__device__ __forceinline__ uint32_t lower_bound(const uint32_t *keys, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// One wavefront per cell: its positions by binary search, then its rows one
// after the other.
template <typename T>
__global__ __launch_bounds__(256) void sums_kernel(const T *__restrict__ grad, uint64_t stride,
                                                   uint32_t width, uint32_t num_cells,
                                                   const uint32_t *__restrict__ keys,
                                                   const uint32_t *__restrict__ index, uint32_t n,
                                                   const float *__restrict__ weight, float scale,
                                                   T *__restrict__ table_grad) {
    const uint64_t v = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    if (v >= num_cells) return;
    const uint32_t lo = lower_bound(keys, n, (uint32_t)v);
    const uint32_t hi = lower_bound(keys, n, (uint32_t)v + 1u);
    for (uint32_t d = threadIdx.x & 63u; d < width; d += 64u) {
        float s = 0.0f;
        for (uint32_t k = lo; k < hi; ++k) {
            const uint32_t i = index[k];
            const float f = weight ? scale * weight[i] : scale;
            s = fmaf(f, (float)grad[(uint64_t)i * stride + d], s);
        }
        table_grad[v * width + d] = (T)s;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void weight_grad_kernel(const T *__restrict__ grad,
                                                          uint64_t grad_stride,
                                                          const T *__restrict__ table,
                                                          uint64_t table_stride, uint32_t num_cells,
                                                          uint32_t width,
                                                          const void *__restrict__ cells,
                                                          int id_type, uint64_t count, float scale,
                                                          float *__restrict__ weight_grad) {
    const uint64_t i = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    if (i >= count) return;
    const int32_t c = load_id(cells, id_type, i, num_cells);
    float s = 0.0f;
    if (c >= 0)
        for (uint32_t d = threadIdx.x & 63u; d < width; d += 64u)
            s = fmaf((float)grad[i * grad_stride + d], (float)table[(uint64_t)c * table_stride + d], s);
    s = group_sum<64>(s);
    if ((threadIdx.x & 63u) == 0) weight_grad[i] = scale * s;
}

size_t align256(size_t x) { return (x + 255u) & ~(size_t)255u; }

int check_rows(const char *what, int type, uint64_t num_cells, int id_type, uint64_t count) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: unknown element type %d", what, type);
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "%s: unknown id type %d", what, id_type);
    if (num_cells >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 cells", what);
    if (count >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 ids", what);
    return SDF_OK;
}

bool misaligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

} // namespace

extern "C" {

int sdf_cell_rows(int type, const void *table, uint64_t table_stride, uint64_t num_cells,
                  uint32_t width, int id_type, const void *cells, uint64_t count,
                  const float *weight, float scale, void *rows, void *stream) {
    const int rc = check_rows("cell_rows", type, num_cells, id_type, count);
    if (rc != SDF_OK) return rc;
    if (count == 0 || width == 0) return SDF_OK;
    if (!cells || !rows || (num_cells > 0 && !table))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    if (misaligned(table, type_bytes(type)) || misaligned(rows, type_bytes(type)))
        return fail(SDF_E_INVALID, "cell_rows: table and rows must be aligned to their elements");
    const uint64_t blocks = (count * width + 255u) / 256u;
    if (blocks > 0x7fffffffull) return fail(SDF_E_INVALID, "cell_rows: too many elements");
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0,
                           static_cast<hipStream_t>(stream), static_cast<const T *>(table),
                           (uint32_t)num_cells, width, table_stride, cells, id_type, count, weight,
                           scale, static_cast<T *>(rows));
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "cell_rows");
}

size_t sdf_cell_rows_backward_scratch_bytes(uint64_t num_cells, uint32_t width, uint64_t count) {
    (void)num_cells;
    (void)width;
    const uint64_t tiles = (count + kTile - 1) / kTile;
    return 4 * align256(4 * count) + align256(4 * tiles * kDigits) + 256;
}

int sdf_cell_rows_backward(int type, const void *rows_grad, uint64_t rows_grad_stride,
                           const void *table, uint64_t table_stride, uint64_t num_cells,
                           uint32_t width, int id_type, const void *cells, uint64_t count,
                           const float *weight, float scale, void *table_grad, float *weight_grad,
                           void *scratch, size_t scratch_bytes, void *stream) {
    const int rc = check_rows("cell_rows_backward", type, num_cells, id_type, count);
    if (rc != SDF_OK) return rc;
    if (!table_grad && !weight_grad) return SDF_OK;
    if ((count > 0 && !cells) ||
        (count > 0 && width > 0 && !rows_grad) || !scratch ||
        (weight_grad && num_cells > 0 && width > 0 && !table))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_cell_rows_backward_scratch_bytes(num_cells, width, count);
    if (scratch_bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    if (misaligned(scratch, 256)) return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t n = (uint32_t)count, tiles = (n + kTile - 1) / kTile;
    char *at = static_cast<char *>(scratch);
    uint32_t *buf[4];
    for (auto &b : buf) {
        b = reinterpret_cast<uint32_t *>(at);
        at += align256(4 * count);
    }
    SortPass p = {cells, id_type, (uint32_t)num_cells, nullptr, nullptr, buf[0], buf[1],
                  reinterpret_cast<uint32_t *>(at), n, tiles, 0};
    const uint32_t *keys = buf[0], *index = buf[1];
    if (table_grad && n > 0) {
        uint32_t k = 0;
        do { // until every bit of the largest key, num_cells, is sorted by
            hipLaunchKernelGGL(sort_count_kernel, dim3(tiles), dim3(256), 0, s, p);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, s, p.counts,
                               tiles * kDigits);
            hipLaunchKernelGGL(sort_scatter_kernel, dim3(tiles), dim3(256), 0, s, p);
            keys = p.keys_out;
            index = p.index_out;
            k ^= 2u;
            p.ids = nullptr;
            p.keys_in = keys;
            p.index_in = index;
            p.keys_out = buf[k];
            p.index_out = buf[k + 1];
            p.shift += 8;
        } while (p.shift < 32 && ((uint32_t)num_cells >> p.shift) != 0);
    }
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (table_grad && num_cells > 0 && width > 0)
            hipLaunchKernelGGL(sums_kernel<T>, dim3((unsigned)((num_cells + 3) / 4)), dim3(256), 0, s,
                               static_cast<const T *>(rows_grad), rows_grad_stride, width,
                               (uint32_t)num_cells, keys, index, n, weight, scale,
                               static_cast<T *>(table_grad));
        if (weight_grad && n > 0)
            hipLaunchKernelGGL(weight_grad_kernel<T>, dim3((unsigned)((count + 3) / 4)), dim3(256),
                               0, s, static_cast<const T *>(rows_grad), rows_grad_stride,
                               static_cast<const T *>(table), table_stride, (uint32_t)num_cells,
                               width, cells, id_type, count, scale, weight_grad);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "cell_rows_backward");
}

} // extern "C"
