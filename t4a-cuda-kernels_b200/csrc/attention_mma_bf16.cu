// The warp-level attention kernels of one cache kind (one file a kind, so that they build beside
// each other).
#include "attention_mma.cuh"
#include "attention_launch.h"

namespace t4a {
namespace cache {

int launch_mma_bf16(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks) {
  return launch_mma<T4A_BF16>(a, padded, row_tiles, stream, blocks);
}

}  // namespace cache
}  // namespace t4a
