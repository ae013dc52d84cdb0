// Host side of the products of rows in groups (products.hip).
#pragma once

#include "product_device.h"

namespace sdfoam_hip {
namespace head {

// How a product is cut: tiles of the result, parts of the inner dimension, and the scratch
// that the parts' sums take.
struct Plan {
    uint64_t tiles;
    uint32_t tiles_n, splits, k_each;
    bool large; // tiles of 256 x 256, else 128 x 128
    uint32_t thin_m, thin_n; // few rows a group: tiles of 16 thin_m x 16 thin_n; 0: not so
    bool late; // the rows' adapters are added when the parts are joined
    size_t bytes;
};
// rows form: rows x n, k summed over, b across k or along it (skinny: tiles of 128 x 32,
// results in fp32)
Plan plan_rows(uint64_t rows, uint32_t groups, bool grouped, uint32_t n, uint32_t k, bool across,
               bool skinny);
// weights form: per group m x n, its rows summed over; narrow: 32 of m (a is fp32) or of n (b is)
Plan plan_weights(uint64_t rows, uint32_t groups, uint32_t m, uint32_t n, bool narrow_m, bool narrow_n);

// the same plan with the adapters added late: where rows have an adapter each, more or less,
// every row's is read by threads of its own
Plan late(Plan plan, uint64_t rows, uint32_t n);

hipError_t product_rows(int type, const ProductArgs &p, const Plan &plan, bool across, bool skinny,
                        bool out_float, hipStream_t s);
hipError_t product_weights(int type, ProductArgs p, const Plan &plan, bool narrow_m, bool narrow_n,
                           hipStream_t s);
int check_blocks(const char *call, const Plan &plan);

} // namespace head
} // namespace sdfoam_hip
