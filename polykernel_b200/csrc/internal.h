// internal.h - what the library's translation units share on the host side.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace pkb200 {
namespace internal {

// Kernel families of pkb200_path_counters.
enum LaunchKind { kAttnTensor = 2, kOther = 4 };

// SM count of the current device and the address of its error word.
int device(int* sms, int** err);
// Opts `func` into `smem` bytes of dynamic shared memory on the current device.
int smem_attr(const void* func, int smem);
// Rank-r tiled map with 128-byte swizzle; dims[0] is the contiguous axis.
bool tensor_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                const cuuint64_t* dims, const cuuint64_t* strides_bytes, const cuuint32_t* box);
void count_launch(LaunchKind kind);

}  // namespace internal
}  // namespace pkb200
