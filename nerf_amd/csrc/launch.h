// Host-side parts of launches that expert_linear.hip and muon.hip share.
#pragma once
#include "nrf_common.h"

namespace nrf {

// Any number of workgroups.  A launch has less than 2^32 work-items along a dimension (more are cut off without an error):
// workgroups past kGridRow, which keeps their deal to the eight XCDs, go on in the next row, a last row's rest past the end.
constexpr int64_t kGridRow = 1 << 22;
inline dim3 grid_rows(int64_t blocks) {
    return blocks <= kGridRow ? dim3(unsigned(blocks)) : dim3(unsigned(kGridRow), unsigned((blocks + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int grid_block() { return int(blockIdx.x + blockIdx.y * unsigned(kGridRow)); }

// whether two tensors (either may be NULL or empty) share memory
inline bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && a_bytes > 0 && b_bytes > 0 && x < y + uintptr_t(b_bytes) && y < x + uintptr_t(a_bytes);
}

}  // namespace nrf
