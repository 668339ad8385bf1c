// Chunked prefill whose queries attend the first n_sink tokens besides their
// sliding window: launches of lnskv_prefill.h's kernel with SINK.
#include "lnskv_prefill.h"

namespace lnskv {

int launch_prefill_mfma_sink(const PrefillArgs& a, int rep, int head_dim, int n_tiles, hipStream_t st) {
  return launch_prefill_kernel<true>(a, rep, head_dim, n_tiles, st);
}

}  // namespace lnskv
