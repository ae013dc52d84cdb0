// Device pieces shared by the label-field kernels (cell_rows.hip,
// label_kernels.hip): element and id types, 16-byte pieces of rows, and sums over
// neighbouring lanes.
#pragma once

#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "../../include/sdfoam_hip.h"

namespace sdfoam_hip {

// sdf_last_error()'s message and `code` (capi.hip)
int fail(int code, const char *fmt, ...);
int hip_fail(hipError_t e, const char *where);

namespace label {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// f(a value of the element type) for SDF_TYPE_*; the caller has checked `type`
template <typename F> inline auto with_type(int type, F f) {
    if (type == SDF_TYPE_F16) return f(half_t());
    if (type == SDF_TYPE_BF16) return f(bf16_t());
    return f(float());
}

inline size_t type_bytes(int type) { return type == SDF_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type >= SDF_TYPE_F32 && type <= SDF_TYPE_BF16; }
inline bool known_id_type(int type) { return type >= SDF_ID_U32 && type <= SDF_ID_I64; }

// The i-th id, or -1 where it does not lie in [0, limit) (limit < 2^31): no
// cell, no label.
__device__ __forceinline__ int32_t load_id(const void *ids, int id_type, uint64_t i,
                                           uint32_t limit) {
    if (id_type == SDF_ID_I64) {
        const uint64_t v = static_cast<const uint64_t *>(ids)[i];
        return v < limit ? (int32_t)v : -1;
    }
    const uint32_t v = static_cast<const uint32_t *>(ids)[i];
    return v < limit ? (int32_t)v : -1;
}

// 16 bytes of a row: kN elements, at any address that the element type allows
// (the hardware takes 16-byte accesses at element alignment).
template <typename T> struct Chunk {
    static constexpr int kN = 16 / (int)sizeof(T);
    T v[kN];
};
template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T *p) {
    Chunk<T> c;
    __builtin_memcpy(&c, p, 16);
    return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T *p, const Chunk<T> &c) {
    __builtin_memcpy(p, &c, 16);
}
// A row's [begin, end) in chunks at begin + k kN.  Only whole chunks inside it
// are read: one that would pass the end is read where it ends there instead
// (place()), and its elements before `at`, which belong to the chunk before it
// (all of them, where `at` is past the end), are set to `fill`.  A range
// shorter than a chunk goes element by element.
template <typename T>
__device__ __forceinline__ uint32_t place(uint32_t at, uint32_t begin, uint32_t end) {
    return end - begin < (uint32_t)Chunk<T>::kN ? at : min(at, end - Chunk<T>::kN);
}
template <typename T>
__device__ __forceinline__ Chunk<T> load_raw(const T *row, uint32_t at, uint32_t begin,
                                             uint32_t end, T fill) {
    if (end - begin >= (uint32_t)Chunk<T>::kN) return load_chunk(row + place<T>(at, begin, end));
    Chunk<T> c;
#pragma unroll
    for (int e = 0; e < Chunk<T>::kN; ++e) c.v[e] = at + e < end ? row[at + e] : fill;
    return c;
}
template <typename T>
__device__ __forceinline__ void mask_chunk(Chunk<T> &c, uint32_t at, uint32_t begin, uint32_t end,
                                           T fill) {
    const uint32_t from = place<T>(at, begin, end);
    if (from == at) return;
#pragma unroll
    for (int e = 0; e < Chunk<T>::kN; ++e)
        if (from + e < at) c.v[e] = fill;
}
// The chunk's own elements into a row (those that mask_chunk leaves).
template <typename T>
__device__ __forceinline__ void store_own(T *row, uint32_t at, uint32_t begin, uint32_t end,
                                          const Chunk<T> &c) {
    if (at + Chunk<T>::kN <= end) {
        store_chunk(row + at, c);
        return;
    }
    const uint32_t from = place<T>(at, begin, end);
#pragma unroll
    for (int e = 0; e < Chunk<T>::kN; ++e)
        if (from + e >= at && from + e < end) row[from + e] = c.v[e];
}

// What a wavefront's lanes wrote to LDS before it, all of them see after it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x of the lane across: lanes of 2, 4, 8 and 16 meet through the VALU's own
// crossbar (quads by xor; eights and sixteens mirrored, which pairs up equal
// values once the smaller steps are done), 32 and 64 through LDS's.
template <int kStep> __device__ __forceinline__ uint32_t across(uint32_t x) {
    if constexpr (kStep == 1) return __builtin_amdgcn_update_dpp(x, x, 0xb1, 0xf, 0xf, false);
    else if constexpr (kStep == 2) return __builtin_amdgcn_update_dpp(x, x, 0x4e, 0xf, 0xf, false);
    else if constexpr (kStep == 4) return __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false);
    else if constexpr (kStep == 8) return __builtin_amdgcn_update_dpp(x, x, 0x140, 0xf, 0xf, false);
    else return (uint32_t)__shfl_xor((int)x, kStep);
}
template <int kStep> __device__ __forceinline__ float across(float x) {
    return __uint_as_float(across<kStep>(__float_as_uint(x)));
}

// op over the kLanes neighbouring lanes (a power of two), in every one of
// them; op must not depend on the order of its arguments.
template <int kLanes, typename V, typename F> __device__ __forceinline__ V group_all(V x, F op) {
    if constexpr (kLanes > 1) x = op(x, across<1>(x));
    if constexpr (kLanes > 2) x = op(x, across<2>(x));
    if constexpr (kLanes > 4) x = op(x, across<4>(x));
    if constexpr (kLanes > 8) x = op(x, across<8>(x));
    if constexpr (kLanes > 16) x = op(x, across<16>(x));
    if constexpr (kLanes > 32) x = op(x, across<32>(x));
    return x;
}
template <int kLanes> __device__ __forceinline__ float group_max(float x) {
    return group_all<kLanes>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int kLanes> __device__ __forceinline__ float group_sum(float x) {
    return group_all<kLanes>(x, [](float a, float b) { return a + b; });
}

} // namespace label
} // namespace sdfoam_hip
