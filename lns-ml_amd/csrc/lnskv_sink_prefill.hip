// Chunked prefill whose queries attend the first n_sink tokens besides their
// sliding window: launches of lnskv_prefill.h's kernel with SINK.
#include "lnskv_prefill.h"

namespace lnskv {

int launch_prefill_mfma_sink(const PrefillArgs& a, int rep, int head_dim, int n_tiles, hipStream_t st) {
  if (int rc = launch_prefill_kernel<true>(a, rep, head_dim, n_tiles, st)) return rc;
  if (a.splits <= 1) return LNSKV_OK;
  const int64_t rows = (int64_t)a.n_tok * a.n_heads;
  const unsigned blocks = (unsigned)((rows + kWavesPerBlock - 1) / kWavesPerBlock);
  if (head_dim == 256)
    prefill_merge_kernel<256><<<blocks, kBlock, 0, st>>>(a);
  else
    prefill_merge_kernel<128><<<blocks, kBlock, 0, st>>>(a);
  return hip_check("prefill merge kernel launch");
}

}  // namespace lnskv
