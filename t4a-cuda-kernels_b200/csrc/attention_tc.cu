// Instances and launches of the tensor-memory attention kernel.
#include "attention_launch.h"
#include "attention_tc.cuh"

namespace t4a {
namespace cache {
namespace {

template <int Kind, int Dim, bool kPasses>
int launch_one_tc(const AttendArgs& a, cudaStream_t stream) {
  static std::atomic<unsigned long long> allowed{0};
  T4A_TRY(runtime::allow_shared(k_attend_tc<Kind, Dim, kPasses>, TcShape<Dim>::shared, &allowed));
  return runtime::launch_early<AttendArgs>(k_attend_tc<Kind, Dim, kPasses>, a.groups * a.row_tiles,
                                           TcRoles<KindOf<Kind>::quantised>::threads, TcShape<Dim>::shared, stream, a);
}

template <int Kind>
int launch_kind_tc(const AttendArgs& a, int padded, cudaStream_t stream) {
  if (padded == 64) return a.passes ? launch_one_tc<Kind, 64, true>(a, stream) : launch_one_tc<Kind, 64, false>(a, stream);
  return a.passes ? launch_one_tc<Kind, 128, true>(a, stream) : launch_one_tc<Kind, 128, false>(a, stream);
}

}  // namespace

int launch_tc(int kind, const AttendArgs& a, int padded, cudaStream_t stream, int* blocks) {
  if (blocks != nullptr) {
    *blocks = kSms * TcShape<128>::per_sm;
    return T4A_OK;
  }
  switch (kind) {
    case T4A_F16: return launch_kind_tc<T4A_F16>(a, padded, stream);
    case T4A_BF16: return launch_kind_tc<T4A_BF16>(a, padded, stream);
    case T4A_I8: return launch_kind_tc<T4A_I8>(a, padded, stream);
    default: return launch_kind_tc<T4A_E4M3>(a, padded, stream);
  }
}

}  // namespace cache
}  // namespace t4a
