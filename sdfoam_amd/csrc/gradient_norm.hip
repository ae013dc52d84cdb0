// The norm of many tensors together, and the tensors scaled to at most a given norm:
//
//   norm   = scale sqrt(sum over all tensors and elements of g^2)
//   factor = scale min(1, max_norm / (norm + 1e-6))        out = factor g
//
// Squares are added in fp64: those of floats below 1e-19 or above 1e19 leave fp32's range,
// and memory is the bound all the same.  The tensors' addresses travel in the launch's
// arguments, kTensors a launch: nothing is copied to the device beforehand, a captured
// graph keeps them.  Every block's share is decided by the sizes alone, and the blocks'
// sums are added in order: every run gives the same.
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
constexpr uint32_t kTensors = 96;
constexpr uint32_t kBlocks = 1024; // a launch
// Up to so many blocks' sums, every block that scales adds them up itself; more are
// added by a launch of their own.
constexpr uint32_t kFewSums = 4096;

struct Tensors {
    const void *in[kTensors];
    void *out[kTensors];
    uint64_t count[kTensors];
    uint32_t chunk[kTensors + 1]; // chunks before each tensor's
    uint8_t type[kTensors], out_type[kTensors];
    uint32_t tensors;
};

struct Piece {
    uint32_t tensor;
    uint64_t first, count;
};
__device__ __forceinline__ Piece piece_of(const Tensors &t, uint32_t chunk) {
    uint32_t lo = 0, hi = t.tensors; // chunk[lo] <= chunk < chunk[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (t.chunk[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    const uint64_t first = (uint64_t)(chunk - t.chunk[lo]) * kChunk;
    const uint64_t left = t.count[lo] - first;
    return {lo, first, left < kChunk ? left : kChunk};
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
    double s = 0.0;
    const uint32_t whole = n / kN;
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < whole; c += kThreads) {
        const Chunk<T> v = load_chunk(p + (uint64_t)c * kN);
#pragma unroll
        for (uint32_t e = 0; e < kN; ++e) s = fma((double)v[e], (double)v[e], s);
    }
    for (uint32_t i = whole * kN + threadIdx.x; i < n; i += kThreads) {
        const double v = (double)(float)p[i];
        s = fma(v, v, s);
    }
    return s;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Tensors t, double *sums) {
    __shared__ double lds[kThreads / 64];
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < t.chunk[t.tensors]; c += gridDim.x) {
        const Piece k = piece_of(t, c);
        const uint32_t n = (uint32_t)k.count;
        if (t.type[k.tensor] == SDF_TYPE_F32) s += squares(static_cast<const float *>(t.in[k.tensor]) + k.first, n);
        else if (t.type[k.tensor] == SDF_TYPE_F16) s += squares(static_cast<const half_t *>(t.in[k.tensor]) + k.first, n);
        else s += squares(static_cast<const bf16_t *>(t.in[k.tensor]) + k.first, n);
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__device__ __forceinline__ double total_of(const double *sums, uint32_t n, double *lds) {
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) s += sums[i];
    return block_sum(s, lds);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double *sums, uint32_t n, float scale,
                                                        float *norm, double *total) {
    __shared__ double lds[kThreads / 64];
    const double s = total_of(sums, n, lds);
    if (threadIdx.x == 0) {
        if (norm) *norm = (float)((double)scale * sqrt(s));
        if (total) *total = s;
    }
}

template <typename T, typename O>
__device__ __forceinline__ void scaled(const T *p, O *o, uint32_t n, float f) {
    constexpr uint32_t kN = Chunk<T>::kN;
    const uint32_t whole = n / kN;
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < whole; c += kThreads) {
        const Chunk<T> v = load_chunk(p + (uint64_t)c * kN);
        O r[kN];
#pragma unroll
        for (uint32_t e = 0; e < kN; ++e) r[e] = (O)(f * v[e]);
        __builtin_memcpy(o + (uint64_t)c * kN, r, sizeof(r));
    }
    for (uint32_t i = whole * kN + threadIdx.x; i < n; i += kThreads) o[i] = (O)(f * (float)p[i]);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Tensors t, const double *sums, uint32_t n,
                                                         float scale, float max_norm, float *norm) {
    __shared__ double lds[kThreads / 64];
    const double size = (double)scale * sqrt(total_of(sums, n, lds));
    double c = (double)max_norm / (size + 1e-6);
    c = c > 1.0 ? 1.0 : c; // NaN stays
    const float f = (float)(scale * c);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)size;
    for (uint32_t c = blockIdx.x; c < t.chunk[t.tensors]; c += gridDim.x) {
        const Piece k = piece_of(t, c);
        const uint32_t count = (uint32_t)k.count;
        const void *in = t.in[k.tensor];
        void *out = t.out[k.tensor];
        if (in == out && f == 1.0f) continue;
        const int type = t.type[k.tensor];
        if (type == SDF_TYPE_F32)
            scaled(static_cast<const float *>(in) + k.first, static_cast<float *>(out) + k.first, count, f);
        else if (t.out_type[k.tensor] == SDF_TYPE_F32) {
            if (type == SDF_TYPE_F16)
                scaled(static_cast<const half_t *>(in) + k.first, static_cast<float *>(out) + k.first, count, f);
            else
                scaled(static_cast<const bf16_t *>(in) + k.first, static_cast<float *>(out) + k.first, count, f);
        } else if (type == SDF_TYPE_F16)
            scaled(static_cast<const half_t *>(in) + k.first, static_cast<half_t *>(out) + k.first, count, f);
        else
            scaled(static_cast<const bf16_t *>(in) + k.first, static_cast<bf16_t *>(out) + k.first, count, f);
    }
}

constexpr uint64_t kMaxElements = 1ull << 40; // of all tensors: 32 bits count the chunks

// kTensors tensors that have elements a launch; f(the tensors, the blocks of the launch).
template <typename F>
hipError_t each_launch(uint32_t n, const int *types, const void *const *in, const int *out_types,
                       void *const *out, const uint64_t *counts, F f) {
    Tensors t;
    t.tensors = 0;
    t.chunk[0] = 0;
    const auto flush = [&]() -> hipError_t {
        if (t.tensors == 0) return hipSuccess;
        const uint32_t chunks = t.chunk[t.tensors];
        f(t, chunks < kBlocks ? chunks : kBlocks);
        t.tensors = 0;
        return hipGetLastError();
    };
    for (uint32_t i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        const uint64_t chunks = (counts[i] + kChunk - 1) / kChunk;
        if (t.tensors == kTensors) {
            const hipError_t e = flush();
            if (e != hipSuccess) return e;
        }
        const uint32_t k = t.tensors++;
        t.in[k] = in[i];
        t.out[k] = out ? out[i] : nullptr;
        t.count[k] = counts[i];
        t.type[k] = (uint8_t)types[i];
        t.out_type[k] = (uint8_t)(out ? out_types[i] : types[i]);
        t.chunk[k + 1] = t.chunk[k] + (uint32_t)chunks;
    }
    return flush();
}

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

uint64_t sums_of(uint32_t n) { return ((uint64_t)n / kTensors + 2) * kBlocks; }

} // namespace

extern "C" {

size_t sdf_clip_gradients_scratch_bytes(uint32_t num_tensors) {
    return round_up((sums_of(num_tensors) + 1) * 8);
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
    const double *from = sums;
    const uint64_t room = sums_of(num_tensors);
    uint32_t n = 0;
    hipError_t e = each_launch(num_tensors, types, gradients, nullptr, nullptr, counts,
                               [&](const Tensors &t, uint32_t blocks) {
                                   squares_kernel<<<blocks, kThreads, 0, s>>>(t, sums + n);
                                   n += blocks;
                               });
    bool said = false;
    if (e == hipSuccess && out && n > 0) {
        if (n > kFewSums) {
            norm_kernel<<<1, kThreads, 0, s>>>(sums, n, scale, nullptr, sums + room);
            from = sums + room;
            n = 1;
        }
        e = each_launch(num_tensors, types, gradients, out_types, out, counts,
                        [&](const Tensors &t, uint32_t blocks) {
                            scale_kernel<<<blocks, kThreads, 0, s>>>(t, from, n, scale, max_norm,
                                                                     said ? nullptr : norm);
                            said = true;
                        });
    }
    if (e == hipSuccess && !said) {
        norm_kernel<<<1, kThreads, 0, s>>>(sums, n, scale, norm, nullptr);
        e = hipGetLastError();
    }
    return e == hipSuccess ? SDF_OK : hip_fail(e, "clip_gradients");
}

} // extern "C"
