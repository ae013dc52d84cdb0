// Device pieces shared by the label-field kernels (cell_rows.hip,
// label_kernels.hip): element and id types, and sums over a wavefront or block.
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

__device__ __forceinline__ float wave_max(float x) {
    for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

} // namespace label
} // namespace sdfoam_hip
