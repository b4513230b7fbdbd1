// Work-groups in two dimensions: a launch takes fewer than 2^32 threads along x.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mogt {

constexpr int WIDE_GRID_LOG2 = 20;
constexpr int64_t WIDE_GRID_MAX = 65535ll << WIDE_GRID_LOG2;

// `groups` work-groups (up to WIDE_GRID_MAX) or some more, numbered by wide_block()
inline dim3 wide_grid(int64_t groups, unsigned z = 1) {
    const int64_t x = groups < (1 << WIDE_GRID_LOG2) ? groups : 1 << WIDE_GRID_LOG2;
    return dim3(static_cast<unsigned>(x), static_cast<unsigned>((groups + x - 1) / x), z);
}
// A second row follows only rows of 2^20: the grid's size is not read.
__device__ __forceinline__ int64_t wide_block() { return static_cast<int64_t>(blockIdx.y) << WIDE_GRID_LOG2 | blockIdx.x; }

}  // namespace mogt
