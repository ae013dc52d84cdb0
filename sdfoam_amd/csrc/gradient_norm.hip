// The norm of many tensors together, and the tensors scaled to at most a given norm:
//
//   norm   = scale sqrt(sum over all tensors and elements of g^2)
//   factor = scale min(1, max_norm / (norm + 1e-6))        out = factor g
//
// Squares are added in fp64: those of floats below 1e-19 or above 1e19 leave fp32's range,
// and memory is the bound all the same.  The tensors' addresses travel in the launches'
// arguments, which a captured graph keeps: those of the two passes themselves, past 96 tensors
// those of small launches that write them to a table on the device first.  Every block's share
// is decided by the sizes alone, and the blocks' sums are added in order: every run gives the
// same.
#include <algorithm>
#include <new>
#include <vector>

#include "head_device.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;
using namespace sdfoam_hip::head;

namespace {

constexpr uint32_t kThreads = 512;
constexpr uint32_t kChunk = 16384; // elements a block takes at a time
constexpr uint32_t kBlocks = 1024; // a launch: four a CU, all of them there at once
constexpr uint32_t kTensors = 96;  // that a launch's arguments hold

constexpr uint32_t kPastChunks = (128u << 20) / 4 / kChunk; // 128 MiB of floats

struct Entry {
    const void *in;
    void *out;
    uint64_t count;
    uint32_t chunk; // chunks before the tensor's
    uint8_t type, out_type;
};
// Few tensors come with the arguments; more are written to a table first, kTensors a launch,
// so that one launch goes over all of them (four launches each way for 300 tensors of 500M
// bf16 elements: 955 us).
struct Few {
    Entry e[kTensors];
    uint32_t tensors, chunks;
};
struct Many {
    const Entry *e;
    uint32_t tensors, chunks;
};
__global__ __launch_bounds__(64) void table_kernel(Few t, Entry *to) {
    for (uint32_t i = threadIdx.x; i < t.tensors; i += 64) to[i] = t.e[i];
}

// f(tensor, first element, elements) for the block's run of chunks, in order or from its end:
// what the last pass read last is then still in the caches.
template <bool kBack, typename Source, typename F>
__device__ __forceinline__ void each_chunk(const Source &t, F f) {
    const uint32_t each = (t.chunks + gridDim.x - 1) / gridDim.x;
    const uint32_t begin = min(blockIdx.x * each, t.chunks), end = min(begin + each, t.chunks);
    if (begin == end) return;
    const uint32_t start = kBack ? end - 1 : begin;
    uint32_t at = 0, hi = t.tensors; // e[at].chunk <= start < e[hi].chunk
    while (hi - at > 1) {
        const uint32_t mid = (at + hi) / 2;
        if (t.e[mid].chunk <= start) at = mid;
        else hi = mid;
    }
    for (uint32_t k = 0; k < end - begin; ++k) {
        const uint32_t c = kBack ? end - 1 - k : begin + k;
        if (kBack)
            while (t.e[at].chunk > c) --at;
        else
            while (at + 1 < t.tensors && t.e[at + 1].chunk <= c) ++at;
        const uint64_t first = (uint64_t)(c - t.e[at].chunk) * kChunk;
        const uint64_t left = t.e[at].count - first;
        f(t.e[at], first, (uint32_t)(left < kChunk ? left : kChunk));
    }
}

__device__ __forceinline__ double block_sum(double x, double *lds) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) x += lds[w];
    return x;
}

template <typename T> __device__ __forceinline__ double squares(const T *p, uint32_t n) {
    constexpr uint32_t kN = Chunk<T>::kN;
    double s[4] = {};
    const uint32_t whole = n / kN;
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < whole; c += kThreads) {
        const Chunk<T> v = load_chunk(p + (uint64_t)c * kN);
#pragma unroll
        for (uint32_t e = 0; e < kN; ++e) s[e % 4] = fma((double)v[e], (double)v[e], s[e % 4]);
    }
    for (uint32_t i = whole * kN + threadIdx.x; i < n; i += kThreads) {
        const double v = (double)(float)p[i];
        s[0] = fma(v, v, s[0]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

template <typename Source> __global__ __launch_bounds__(kThreads) void squares_kernel(Source t, double *sums) {
    __shared__ double lds[kThreads / 64];
    double s = 0.0;
    each_chunk<false>(t, [&](const Entry &k, uint64_t first, uint32_t n) {
        if (k.type == SDF_TYPE_F32) s += squares(static_cast<const float *>(k.in) + first, n);
        else if (k.type == SDF_TYPE_F16) s += squares(static_cast<const half_t *>(k.in) + first, n);
        else s += squares(static_cast<const bf16_t *>(k.in) + first, n);
    });
    s = block_sum(s, lds);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__device__ __forceinline__ double total_of(const double *sums, uint32_t n, double *lds) {
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) s += sums[i];
    return block_sum(s, lds);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double *sums, uint32_t n, float scale, float *norm) {
    __shared__ double lds[kThreads / 64];
    const double s = total_of(sums, n, lds);
    if (threadIdx.x == 0) *norm = (float)((double)scale * sqrt(s));
}

// 16 bytes of the result a thread, so that a wavefront writes whole lines; large results past
// the caches.
template <typename T, typename O, typename Times>
__device__ __forceinline__ void scaled(const void *in, void *out, uint64_t first, uint32_t n, Times times, bool past) {
    constexpr uint32_t kN = 16 / sizeof(O);
    struct In {
        T v[kN];
    };
    struct Out {
        O v[kN];
    };
    const T *p = static_cast<const T *>(in) + first;
    O *o = static_cast<O *>(out) + first;
    // whole pieces begin where the result's 128 bytes do
    const uint32_t head = min(n, (uint32_t)(-reinterpret_cast<uintptr_t>(o) & 127u) / (uint32_t)sizeof(O));
    if (threadIdx.x < head) o[threadIdx.x] = (O)times((float)p[threadIdx.x]);
    p += head, o += head, n -= head;
    const uint32_t whole = n / kN;
    const auto go = [&](auto store) {
#pragma unroll 4
        for (uint32_t c = threadIdx.x; c < whole; c += kThreads) {
            In v;
            __builtin_memcpy(&v, p + (uint64_t)c * kN, sizeof(v));
            Out r;
#pragma unroll
            for (uint32_t e = 0; e < kN; ++e) r.v[e] = (O)times((float)v.v[e]);
            store(o + (uint64_t)c * kN, r);
        }
    };
    if (past) go([](O *to, const Out &r) { store_past<sizeof(O)>(to, r); });
    else go([](O *to, const Out &r) { __builtin_memcpy(to, &r, sizeof(r)); });
    for (uint32_t i = whole * kN + threadIdx.x; i < n; i += kThreads) o[i] = (O)times((float)p[i]);
}

// Every block adds the other pass's sums itself, in the same order (8 KB from L2).  Memory
// bounds both passes: 500M bf16 elements into floats 165 us (6.1 TB/s) and 604 (5.0); with the
// results written through the caches 210 and 615, unaligned besides 214 and 622.
template <typename Source>
__global__ __launch_bounds__(kThreads) void scale_kernel(Source t, const double *sums, uint32_t n, float scale,
                                                         float max_norm, float *norm) {
    __shared__ double lds[kThreads / 64];
    const double size = (double)scale * sqrt(total_of(sums, n, lds));
    double c = (double)max_norm / (size + 1e-6);
    c = c > 1.0 ? 1.0 : c; // NaN stays
    const double wide = (double)scale * c;
    const float f = (float)wide;
    const bool past = t.chunks >= kPastChunks;
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)size;
    const auto go = [&](auto times) {
        each_chunk<true>(t, [&](const Entry &k, uint64_t first, uint32_t n) {
            if (k.in == k.out && f == 1.0f) return;
            if (k.type == SDF_TYPE_F32) scaled<float, float>(k.in, k.out, first, n, times, past);
            else if (k.type == SDF_TYPE_F16) {
                if (k.out_type == SDF_TYPE_F32) scaled<half_t, float>(k.in, k.out, first, n, times, past);
                else scaled<half_t, half_t>(k.in, k.out, first, n, times, past);
            } else if (k.out_type == SDF_TYPE_F32) scaled<bf16_t, float>(k.in, k.out, first, n, times, past);
            else scaled<bf16_t, bf16_t>(k.in, k.out, first, n, times, past);
        });
    };
    // A factor below fp32's normal range keeps few of its bits there, or none, and gradients
    // of up to 3e38 lift its products back into the range: those in fp64.
    if (wide > 0.0 && wide < 0x1p-126) go([wide](float g) { return (float)(wide * (double)g); });
    else go([f](float g) { return f * g; });
}

constexpr uint64_t kMaxElements = 1ull << 40; // of all tensors: 32 bits count the chunks

int check_tensors(uint32_t n, const int *types, const void *const *in, const uint64_t *counts) {
    if (n > 0 && (!types || !in || !counts)) return fail(SDF_E_INVALID, "NULL pointer argument");
    uint64_t all = 0;
    for (uint32_t i = 0; i < n; ++i) {
        if (!known_type(types[i])) return fail(SDF_E_INVALID, "types must be SDF_TYPE_*");
        if (counts[i] >= kMaxElements || (all += counts[i]) >= kMaxElements)
            return fail(SDF_E_INVALID, "tensors of fewer than 2^40 elements in all");
        if (counts[i] > 0 && !in[i]) return fail(SDF_E_INVALID, "NULL pointer argument");
    }
    return SDF_OK;
}

// Each result lies by itself: on no other, and on no input but its own, from the start.
int check_apart(uint32_t n, const int *types, const void *const *in, const int *out_types,
                void *const *out, const uint64_t *counts) {
    struct Range {
        uintptr_t begin, end;
    };
    std::vector<Range> results;
    results.reserve(n);
    for (uint32_t i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        if (!out[i]) return fail(SDF_E_INVALID, "NULL pointer argument");
        if (out_types[i] != types[i] && out_types[i] != SDF_TYPE_F32)
            return fail(SDF_E_INVALID, "out must be float32 or of the gradient's type");
        if (in[i] == out[i] && out_types[i] != types[i])
            return fail(SDF_E_INVALID, "out must not overlap a gradient of another type");
        const uintptr_t b = reinterpret_cast<uintptr_t>(out[i]);
        results.push_back({b, b + counts[i] * type_bytes(out_types[i])});
    }
    std::sort(results.begin(), results.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    for (size_t k = 1; k < results.size(); ++k)
        if (results[k].begin < results[k - 1].end)
            return fail(SDF_E_INVALID, "the same gradient is there twice, or results overlap");
    for (uint32_t i = 0; i < n; ++i) {
        if (counts[i] == 0 || in[i] == out[i]) continue;
        const uintptr_t b = reinterpret_cast<uintptr_t>(in[i]), e = b + counts[i] * type_bytes(types[i]);
        const auto at = std::upper_bound(results.begin(), results.end(), b,
                                         [](uintptr_t v, const Range &r) { return v < r.end; });
        if (at != results.end() && at->begin < e)
            return fail(SDF_E_INVALID, "out must not overlap another gradient");
    }
    return SDF_OK;
}

template <typename Source>
hipError_t run(const Source &t, bool scales, float max_norm, float scale, float *norm, double *sums,
               hipStream_t s) {
    const uint32_t blocks = t.chunks < kBlocks ? t.chunks : kBlocks;
    if (blocks > 0) squares_kernel<<<blocks, kThreads, 0, s>>>(t, sums);
    if (scales && blocks > 0) scale_kernel<<<blocks, kThreads, 0, s>>>(t, sums, blocks, scale, max_norm, norm);
    else norm_kernel<<<1, kThreads, 0, s>>>(sums, blocks, scale, norm);
    return hipGetLastError();
}

} // namespace

extern "C" {

size_t sdf_clip_gradients_scratch_bytes(uint32_t num_tensors) {
    return round_up(kBlocks * 8) + (num_tensors > kTensors ? round_up((size_t)num_tensors * sizeof(Entry)) : 0);
}

int sdf_clip_gradients(uint32_t num_tensors, const int *types, const void *const *gradients,
                       const uint64_t *counts, const int *out_types, void *const *out,
                       float max_norm, float scale, float *norm, void *scratch,
                       size_t scratch_bytes, void *stream) {
    int rc = check_tensors(num_tensors, types, gradients, counts);
    if (rc != SDF_OK) return rc;
    if (!norm) return fail(SDF_E_INVALID, "NULL pointer argument");
    if (!(scale > 0.0f && scale <= 3.0e38f)) return fail(SDF_E_INVALID, "scale must be positive and finite");
    if (out) {
        if (!(max_norm >= 0.0f)) return fail(SDF_E_INVALID, "max_norm must not be negative");
        if (num_tensors > 0 && !out_types) return fail(SDF_E_INVALID, "NULL pointer argument");
        try {
            rc = check_apart(num_tensors, types, gradients, out_types, out, counts);
        } catch (const std::bad_alloc &) {
            rc = fail(SDF_E_INVALID, "no memory for the check of %u tensors", num_tensors);
        }
        if (rc != SDF_OK) return rc;
    }
    if ((rc = check_scratch(scratch, scratch_bytes, sdf_clip_gradients_scratch_bytes(num_tensors))) != SDF_OK)
        return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    double *sums = static_cast<double *>(scratch);
    Entry *table = reinterpret_cast<Entry *>(static_cast<char *>(scratch) + round_up(kBlocks * 8));
    Few t;
    t.tensors = 0;
    uint32_t chunks = 0, written = 0;
    hipError_t e = hipSuccess;
    for (uint32_t i = 0; i < num_tensors && e == hipSuccess; ++i) {
        if (counts[i] == 0) continue;
        if (t.tensors == kTensors) {
            table_kernel<<<1, 64, 0, s>>>(t, table + written);
            e = hipGetLastError();
            written += kTensors;
            t.tensors = 0;
        }
        t.e[t.tensors++] = {gradients[i], out ? out[i] : nullptr, counts[i], chunks, (uint8_t)types[i],
                            (uint8_t)(out ? out_types[i] : types[i])};
        chunks += (uint32_t)((counts[i] + kChunk - 1) / kChunk);
    }
    t.chunks = chunks;
    if (e == hipSuccess && written > 0) {
        table_kernel<<<1, 64, 0, s>>>(t, table + written);
        e = hipGetLastError();
        if (e == hipSuccess)
            e = run(Many{table, written + t.tensors, chunks}, out != nullptr, max_norm, scale, norm, sums, s);
    } else if (e == hipSuccess) {
        e = run(t, out != nullptr, max_norm, scale, norm, sums, s);
    }
    return e == hipSuccess ? SDF_OK : hip_fail(e, "clip_gradients");
}

} // extern "C"
