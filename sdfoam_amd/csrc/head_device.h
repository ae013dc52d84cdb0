// Pieces shared by the kernels of label fields' heads (expert_rows.hip, products.hip,
// adapters.hip).
#pragma once

#include "label_device.h"

namespace sdfoam_hip {
namespace head {

inline size_t round_up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

inline int check_scratch(const void *scratch, size_t bytes, size_t need) {
    if (need == 0) return SDF_OK;
    if (!scratch || bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, bytes);
    if ((reinterpret_cast<uintptr_t>(scratch) & 255u) != 0)
        return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    return SDF_OK;
}

// The order of n ids by group (expert_rows.hip): places, the entry at each place, its
// group (-1 for none), each NULL where it is not wanted, and offsets [groups + 1].
size_t order_scratch_bytes(uint64_t n, uint32_t groups);
hipError_t launch_order(int id_type, const void *ids, uint64_t n, uint32_t groups,
                        int32_t *places, int32_t *entries, int32_t *group_of, int32_t *offsets,
                        void *scratch, hipStream_t s);

} // namespace head
} // namespace sdfoam_hip
