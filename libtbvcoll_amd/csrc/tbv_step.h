// Shared by the operators of the layer around the all-reduce (tbv_i8rows.hip, tbv_matmul.hip, tbv_rotary.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace tbv {

// A launch dimension holds fewer than 2^32 threads: blocks beyond 2^20 continue in the grid's y (2^20 is a multiple of
// eight, so neighbouring blocks go to the XCDs in turn in either form).
inline dim3 flat_grid(size_t blocks)
{
    const size_t x = blocks < ((size_t)1 << 20) ? blocks : (size_t)1 << 20;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
[[maybe_unused]] static __device__ __forceinline__ size_t flat_block() { return (size_t)blockIdx.y * gridDim.x + blockIdx.x; }

}  // namespace tbv
