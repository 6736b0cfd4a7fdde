// Launches of any number of workgroups.  A launch has less than 2^32 work-items along a dimension: workgroups past kGridRow (which
// keeps their deal to the eight XCDs) go on in the next row, a last row's rest past the end.
#pragma once
#include "nrf_common.h"

namespace nrf {

constexpr int64_t kGridRow = 1 << 22;
inline dim3 grid_rows(int64_t blocks) {
    return blocks <= kGridRow ? dim3(unsigned(blocks)) : dim3(unsigned(kGridRow), unsigned((blocks + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int grid_block() { return int(blockIdx.x + blockIdx.y * unsigned(kGridRow)); }

}  // namespace nrf
