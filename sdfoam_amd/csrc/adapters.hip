// A shared projection with low-rank adapters of the rows' own beside it:
//
//   h_i   = s down_a x_i                (a: the adapter of row i; none: 0)
//   out_i = weight x_i + up_a h_i
//
// and, with b_i = s up_a^T out_grad_i,
//
//   x_grad_i    = weight^T out_grad_i + down_a^T b_i
//   weight_grad = sum_i out_grad_i x_i^T
//   down_grad_a = sum over i of a of b_i x_i^T
//   up_grad_a   = sum over i of a of out_grad_i h_i^T
//
// The rows are put in the order of their adapters (as indices: they are read and written
// where they lie), h and b are products of rows in groups, and the shared product adds
// what its rows' adapters give before it rounds.  h and b stay in fp32.
#include "products.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;
using namespace sdfoam_hip::head;

namespace {

// h of few rows, in the order they come: a wave for each of a row's values.  Bound by its
// chain of loads: 64 rows of 2,048 bf16 and rank 16 6.3 us, one of 4,096 9 (the products in
// parts, with the order before them, took 30 of a call's 35).  A whole call in microseconds
// this way and with the order, 2,048 -> 2,048 bf16 and rank 16: 64 rows of 64 adapters 18 and
// 28, of 8 adapters 57 and 67; 96 rows 21 and 31, 71 and 48.
struct FewRows {
    const void *rows, *ids, *down;
    uint64_t stride;
    int id_type;
    uint32_t width, adapters, rank, pitch;
    float scale;
    float *inner;
    int32_t *group_of;
};
constexpr uint32_t kFewRows = 64;

template <typename T> __global__ __launch_bounds__(256) void few_rows_kernel(FewRows f) {
    constexpr uint32_t kC = Chunk<T>::kN;
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 63u, r = blockIdx.y * 4 + (threadIdx.x >> 6);
    const int32_t a = load_id(f.ids, f.id_type, row, f.adapters);
    if (blockIdx.y == 0 && threadIdx.x == 0) f.group_of[row] = a;
    float sum = 0.0f;
    if (a >= 0 && r < f.rank) {
        const T *x = static_cast<const T *>(f.rows) + row * f.stride;
        const T *d = static_cast<const T *>(f.down) + ((uint64_t)a * f.rank + r) * f.width;
#pragma unroll 4
        for (uint32_t k = lane * kC; k < f.width; k += 64 * kC) {
            const uint32_t have = f.width - k;
            const Few<T, kC> u = load_some<T, kC>(x + k, have), v = load_some<T, kC>(d + k, have);
#pragma unroll
            for (uint32_t e = 0; e < kC; ++e) sum = fmaf((float)u.v[e], (float)v.v[e], sum);
        }
    }
    sum = group_sum<64>(sum);
    // 0 past the rank, at any scale
    if (lane == 0 && r < f.pitch) f.inner[row * f.pitch + r] = r < f.rank ? f.scale * sum : 0.0f;
}

struct Layout {
    size_t order, entries, group_of, offsets, inner, back, partial, bytes;
    uint32_t pitch;
    Plan inner_plan, back_plan, out_plan, rows_plan, down_plan, up_plan, weight_plan;
};

struct Sizes {
    uint64_t count;
    uint32_t width, out_width, adapters, rank;
    bool beside() const { return count > 0 && adapters > 0 && rank > 0; }
};

// Few rows for each adapter, and few enough that their sums in fp32 cost little.  A call's
// microseconds with the adapters added late and in the tiles, 2,048 -> 32,768 bf16 and rank
// 16: 200 rows of 200 adapters 154 and 184, of 25 adapters 134 and 161, of 12 adapters 134 and
// 65; 2,048 -> 8,192: 1,000 rows of 125 adapters 160 and 168, 2,000 of 500 308 and 320.
bool one_each(const Sizes &z) { return z.count <= 1024 && z.count < 8ull * z.adapters; }

bool few(const Sizes &z, bool backward) { return !backward && z.count <= kFewRows; }

Layout layout(const Sizes &z, bool backward) {
    Layout l = {};
    size_t at = 0, partial = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes);
        return here;
    };
    const auto also = [&](const Plan &p) {
        if (p.bytes > partial) partial = p.bytes;
    };
    if (z.beside() && few(z, backward)) {
        l.pitch = (z.rank + 15) / 16 * 16;
        l.group_of = take(z.count * 4);
        l.inner = take(z.count * l.pitch * 4);
    } else if (z.beside()) {
        l.pitch = (z.rank + 15) / 16 * 16;
        l.order = take(order_scratch_bytes(z.count, z.adapters));
        l.entries = take(z.count * 4);
        l.group_of = take(z.count * 4);
        l.offsets = take((z.adapters + 1ull) * 4);
        l.inner = take(z.count * l.pitch * 4);
        also(l.inner_plan = plan_rows(z.count, z.adapters, true, l.pitch, z.width, false, true));
        if (backward) {
            l.back = take(z.count * l.pitch * 4);
            also(l.back_plan = plan_rows(z.count, z.adapters, true, l.pitch, z.out_width, true, true));
            also(l.down_plan = plan_weights(z.count, z.adapters, z.rank, z.width, true, false));
            also(l.up_plan = plan_weights(z.count, z.adapters, z.out_width, z.rank, false, true));
        }
    }
    const auto product = [&](uint32_t n, uint32_t k, bool across) {
        const Plan plan = plan_rows(z.count, 1, false, n, k, across, false);
        return z.beside() && one_each(z) ? late(plan, z.count, n) : plan;
    };
    if (backward) {
        also(l.rows_plan = product(z.width, z.out_width, true));
        also(l.weight_plan = plan_weights(z.count, 1, z.out_width, z.width, false, false));
    } else {
        also(l.out_plan = product(z.out_width, z.width, false));
    }
    l.partial = take(partial);
    l.bytes = at;
    return l;
}

bool fits(const Sizes &z) {
    return z.count < 1ull << 31 && z.adapters <= SDF_MAX_ADAPTERS && z.rank <= SDF_MAX_RANK &&
           z.width <= 1u << 18 && z.out_width <= 1u << 18;
}

int check_sizes(const char *call, int type, int id_type, const Sizes &z) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: type must be SDF_TYPE_*", call);
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "id_type must be SDF_ID_*");
    if (z.adapters > SDF_MAX_ADAPTERS)
        return fail(SDF_E_INVALID, "at most %u adapters (got %u)", SDF_MAX_ADAPTERS, z.adapters);
    if (z.rank > SDF_MAX_RANK)
        return fail(SDF_E_INVALID, "adapters of rank at most %u (got %u)", SDF_MAX_RANK, z.rank);
    if (z.count >= 1ull << 31) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 rows", call);
    if (z.width > 1u << 18 || z.out_width > 1u << 18)
        return fail(SDF_E_INVALID, "%s takes rows of at most 2^18 elements", call);
    return SDF_OK;
}

// the rows' order and what it lies in
struct Ordered {
    int32_t *entries, *group_of, *offsets;
    float *inner, *back, *partial;
    Groups groups;
};

hipError_t order_rows(const Layout &l, const Sizes &z, int id_type, const void *ids, char *scratch,
                      Ordered &o, hipStream_t s) {
    o = {};
    o.partial = reinterpret_cast<float *>(scratch + l.partial);
    if (!z.beside()) return hipSuccess;
    o.entries = reinterpret_cast<int32_t *>(scratch + l.entries);
    o.group_of = reinterpret_cast<int32_t *>(scratch + l.group_of);
    o.offsets = reinterpret_cast<int32_t *>(scratch + l.offsets);
    o.inner = reinterpret_cast<float *>(scratch + l.inner);
    o.back = reinterpret_cast<float *>(scratch + l.back);
    o.groups = {o.offsets, z.adapters, (uint32_t)z.count};
    return launch_order(id_type, ids, z.count, z.adapters, nullptr, o.entries, o.group_of, o.offsets,
                        scratch + l.order, s);
}

// h (down, along its rows) or b (up, across): in the rows' order
hipError_t low_rank(int type, const Plan &plan, const Sizes &z, const Ordered &o, const Layout &l,
                    const void *rows, uint64_t stride, uint32_t k, const void *matrix, bool across,
                    float scale, float *to, hipStream_t s) {
    ProductArgs p = {};
    p.a = {rows, stride, 0, o.entries};
    p.b = {matrix, across ? z.rank : k, (uint64_t)z.rank * k, nullptr};
    p.groups = o.groups;
    p.n = z.rank;
    p.n_out = l.pitch;
    p.k = k;
    p.out = to;
    p.out_stride = l.pitch;
    p.partial = o.partial;
    p.scale = scale;
    return product_rows(type, p, plan, across, true, true, s);
}

} // namespace

extern "C" {

size_t sdf_adapter_linear_scratch_bytes(uint64_t count, uint32_t width, uint32_t out_width,
                                        uint32_t num_adapters, uint32_t rank) {
    const Sizes z = {count, width, out_width, num_adapters, rank};
    return fits(z) ? layout(z, false).bytes : 0;
}

int sdf_adapter_linear(int type, const void *rows, uint64_t rows_stride, uint64_t count,
                       uint32_t width, uint32_t out_width, const void *weight,
                       uint64_t weight_stride, int id_type, const void *adapters,
                       uint32_t num_adapters, uint32_t rank, const void *down, const void *up,
                       float scale, void *out, void *scratch, size_t scratch_bytes, void *stream) {
    const Sizes z = {count, width, out_width, num_adapters, rank};
    int rc = check_sizes("sdf_adapter_linear", type, id_type, z);
    if (rc != SDF_OK) return rc;
    if (count == 0 || out_width == 0) return SDF_OK;
    if (!out || !adapters || (width > 0 && (!rows || !weight || (z.beside() && !down))) || (z.beside() && !up))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const Layout l = layout(z, false);
    if ((rc = check_scratch(scratch, scratch_bytes, l.bytes)) != SDF_OK) return rc;
    for (const Plan *plan : {&l.inner_plan, &l.out_plan})
        if ((rc = check_blocks("sdf_adapter_linear", *plan)) != SDF_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Ordered o = {};
    hipError_t e = hipSuccess;
    if (z.beside() && few(z, false)) {
        char *at = static_cast<char *>(scratch);
        o.inner = reinterpret_cast<float *>(at + l.inner);
        o.group_of = reinterpret_cast<int32_t *>(at + l.group_of);
        o.partial = reinterpret_cast<float *>(at + l.partial);
        const FewRows f = {rows, adapters, down, rows_stride, id_type, width, num_adapters, rank, l.pitch,
                           scale, o.inner, o.group_of};
        const dim3 grid((uint32_t)count, l.pitch / 4);
        with_type(type, [&](auto t) { few_rows_kernel<decltype(t)><<<grid, 256, 0, s>>>(f); });
        e = hipGetLastError();
    } else {
        e = order_rows(l, z, id_type, adapters, static_cast<char *>(scratch), o, s);
        if (e == hipSuccess && z.beside())
            e = low_rank(type, l.inner_plan, z, o, l, rows, rows_stride, width, down, false, scale, o.inner, s);
    }
    if (e == hipSuccess) {
        ProductArgs p = {};
        p.a = {rows, rows_stride, 0, o.entries};
        p.b = {weight, weight_stride, 0, nullptr};
        p.groups = {nullptr, 1, (uint32_t)count};
        p.n = out_width;
        p.k = width;
        p.out = out;
        p.out_stride = out_width;
        p.out_index = o.entries;
        p.partial = o.partial;
        p.scale = 1.0f;
        if (z.beside()) p.beside = {o.inner, rank, l.pitch, up, (uint64_t)out_width * rank, rank, o.group_of};
        e = product_rows(type, p, l.out_plan, false, false, false, s);
    }
    return e == hipSuccess ? SDF_OK : hip_fail(e, "adapter_linear");
}

size_t sdf_adapter_linear_backward_scratch_bytes(uint64_t count, uint32_t width, uint32_t out_width,
                                                 uint32_t num_adapters, uint32_t rank) {
    const Sizes z = {count, width, out_width, num_adapters, rank};
    return fits(z) ? layout(z, true).bytes : 0;
}

int sdf_adapter_linear_backward(int type, const void *out_grad, uint64_t out_grad_stride,
                                const void *rows, uint64_t rows_stride, uint64_t count,
                                uint32_t width, uint32_t out_width, const void *weight,
                                uint64_t weight_stride, int id_type, const void *adapters,
                                uint32_t num_adapters, uint32_t rank, const void *down,
                                const void *up, float scale, void *rows_grad, void *weight_grad,
                                void *down_grad, void *up_grad, void *scratch,
                                size_t scratch_bytes, void *stream) {
    const Sizes z = {count, width, out_width, num_adapters, rank};
    int rc = check_sizes("sdf_adapter_linear_backward", type, id_type, z);
    if (rc != SDF_OK) return rc;
    const bool want_rows = rows_grad && count > 0 && width > 0;
    const bool want_weight = weight_grad && width > 0 && out_width > 0;
    const bool some = num_adapters > 0 && rank > 0;
    const bool want_down = down_grad && some && width > 0, want_up = up_grad && some && out_width > 0;
    if (!want_rows && !want_weight && !want_down && !want_up) return SDF_OK;
    if (count > 0) {
        const bool need_back = z.beside() && (want_rows || want_down);
        if (!adapters || (out_width > 0 && (!out_grad || (want_rows && !weight) || (need_back && !up))) ||
            ((want_weight || want_down || (want_up && width > 0)) && !rows) ||
            (width > 0 && z.beside() && (want_rows || want_up) && !down))
            return fail(SDF_E_INVALID, "NULL pointer argument");
    }
    const Layout l = layout(z, true);
    if ((rc = check_scratch(scratch, scratch_bytes, l.bytes)) != SDF_OK) return rc;
    for (const Plan *plan : {&l.inner_plan, &l.back_plan, &l.rows_plan, &l.weight_plan, &l.down_plan, &l.up_plan})
        if ((rc = check_blocks("sdf_adapter_linear_backward", *plan)) != SDF_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Ordered o = {};
    hipError_t e = hipSuccess;
    if (want_rows || want_down || want_up)
        e = order_rows(l, z, id_type, adapters, static_cast<char *>(scratch), o, s);
    else
        o.partial = reinterpret_cast<float *>(static_cast<char *>(scratch) + l.partial);
    if (e == hipSuccess && z.beside() && (want_rows || want_down))
        e = low_rank(type, l.back_plan, z, o, l, out_grad, out_grad_stride, out_width, up, true, scale, o.back, s);
    if (e == hipSuccess && z.beside() && want_up)
        e = low_rank(type, l.inner_plan, z, o, l, rows, rows_stride, width, down, false, scale, o.inner, s);
    if (e == hipSuccess && want_rows) {
        ProductArgs p = {};
        p.a = {out_grad, out_grad_stride, 0, o.entries};
        p.b = {weight, weight_stride, 0, nullptr};
        p.groups = {nullptr, 1, (uint32_t)count};
        p.n = width;
        p.k = out_width;
        p.out = rows_grad;
        p.out_stride = width;
        p.out_index = o.entries;
        p.partial = o.partial;
        p.scale = 1.0f;
        if (z.beside()) p.beside = {o.back, rank, l.pitch, down, (uint64_t)width * rank, width, o.group_of};
        e = product_rows(type, p, l.rows_plan, true, false, false, s);
    }
    ProductArgs p = {};
    p.groups = o.groups;
    if (!z.beside()) p.groups = {nullptr, num_adapters, 0}; // no rows: gradients of 0
    p.partial = o.partial;
    p.scale = 1.0f;
    if (e == hipSuccess && want_down) {
        p.a = {o.back, l.pitch, 0, nullptr};
        p.b = {rows, rows_stride, 0, o.entries};
        p.m = rank;
        p.n = p.out_stride = width;
        p.out = down_grad;
        e = product_weights(type, p, z.beside() ? l.down_plan : plan_weights(0, num_adapters, rank, width, true, false),
                            true, false, s);
    }
    if (e == hipSuccess && want_up) {
        p.a = {out_grad, out_grad_stride, 0, o.entries};
        p.b = {o.inner, l.pitch, 0, nullptr};
        p.m = out_width;
        p.n = p.out_stride = rank;
        p.out = up_grad;
        e = product_weights(type, p, z.beside() ? l.up_plan : plan_weights(0, num_adapters, out_width, rank, false, true),
                            false, true, s);
    }
    if (e == hipSuccess && want_weight) {
        p.a = {out_grad, out_grad_stride, 0, nullptr};
        p.b = {rows, rows_stride, 0, nullptr};
        p.groups = {nullptr, 1, (uint32_t)count};
        p.m = out_width;
        p.n = p.out_stride = width;
        p.out = weight_grad;
        e = product_weights(type, p, l.weight_plan, false, false, s);
    }
    return e == hipSuccess ? SDF_OK : hip_fail(e, "adapter_linear_backward");
}

} // extern "C"
