// Launches of k_attend for one cache kind: the padded dim and the row tiles pick the instance.
#pragma once

#include "attention_mma.cuh"
#include "runtime.h"

namespace t4a {
namespace cache {

constexpr int kSms = 148;

// The most tiles of 8 query rows that the warp-level kernel takes at once; the rule's reasons are
// where the kernel is chosen.
constexpr int most_row_tiles(bool quantised, int padded) {
  if (padded == 256) return 2;
  if (quantised) return 4;
  return padded == 128 ? 1 : 2;
}

// With `blocks`, only says how many blocks to launch: as many as the SMs hold at once.
template <int Kind, int Dim, int kRowTiles>
int launch_one(const AttendArgs& a, cudaStream_t stream, int* blocks) {
  using Shape = MmaShape<Kind, Dim, kRowTiles>;
  if (blocks != nullptr) {
    *blocks = kSms * Shape::per_sm;
    return T4A_OK;
  }
  static std::atomic<unsigned long long> allowed{0};
  T4A_TRY(runtime::allow_shared(k_attend<Kind, Dim, kRowTiles>, Shape::shared, &allowed));
  return runtime::launch_early<AttendArgs>(k_attend<Kind, Dim, kRowTiles>, a.groups * a.row_tiles, kMmaThreads,
                                           Shape::shared, stream, a);
}

template <int Kind, int Dim>
int launch_rows_of(const AttendArgs& a, int row_tiles, cudaStream_t stream, int* blocks) {
  constexpr int kMost = most_row_tiles(KindOf<Kind>::quantised, Dim);
  if (row_tiles == 1) return launch_one<Kind, Dim, 1>(a, stream, blocks);
  if constexpr (kMost >= 2)
    if (row_tiles == 2) return launch_one<Kind, Dim, 2>(a, stream, blocks);
  if constexpr (kMost >= 4)
    if (row_tiles == 4) return launch_one<Kind, Dim, 4>(a, stream, blocks);
  return T4A_ERR_UNSUPPORTED_OP;
}

template <int Kind>
int launch_mma(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks) {
  switch (padded) {
    case 64: return launch_rows_of<Kind, 64>(a, row_tiles, stream, blocks);
    case 96: return launch_rows_of<Kind, 96>(a, row_tiles, stream, blocks);
    case 128: return launch_rows_of<Kind, 128>(a, row_tiles, stream, blocks);
    default: return launch_rows_of<Kind, 256>(a, row_tiles, stream, blocks);
  }
}

constexpr int kTcTileRows = 128;  // rows of a unit in the tensor-memory kernel
int launch_tc(int kind, const AttendArgs& a, int padded, cudaStream_t stream, int* blocks);

int launch_mma_f16(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks);
int launch_mma_bf16(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks);
int launch_mma_i8(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks);
int launch_mma_e4m3(const AttendArgs& a, int padded, int row_tiles, cudaStream_t stream, int* blocks);

}  // namespace cache
}  // namespace t4a
