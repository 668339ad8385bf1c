// Chunked prefill without sinks: launches of lnskv_prefill.h's kernel.
#include "lnskv_prefill.h"

namespace lnskv {
namespace {

template <int NH>
int prefill_qt(int rep) {
  switch (rep) {
    case 1: return PfShape<1, NH>::QT;
    case 2: return PfShape<2, NH>::QT;
    case 4: return PfShape<4, NH>::QT;
    default: return PfShape<8, NH>::QT;
  }
}
}  // namespace

int prefill_queries_per_tile(int rep, int head_dim) {
  return head_dim == 256 ? prefill_qt<2>(rep) : prefill_qt<1>(rep);
}

int launch_prefill_mfma(const PrefillArgs& a, int rep, int head_dim, int n_tiles, hipStream_t st) {
  return launch_prefill_kernel<false>(a, rep, head_dim, n_tiles, st);
}

}  // namespace lnskv
