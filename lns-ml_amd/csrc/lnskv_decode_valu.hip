// Launchers of the generic decode kernel (lnskv_decode_valu.h) over the window
// [p_start, kv_len) of every sequence.
#include "lnskv_decode_valu.h"

namespace lnskv {

template <int DT, int D, int REP, bool FUSED>
static void launch_t(const DecodeArgs& a, int n_seq, hipStream_t st) {
  const dim3 grid((unsigned)a.n_kv, (unsigned)a.max_parts, (unsigned)n_seq);
  decode_valu_kernel<DT, D, REP, FUSED><<<grid, kBlock, 0, st>>>(a);
  launch_combine<REP, D, FUSED>(a, n_seq, st);
}

template <int DT, int D, bool FUSED>
static int launch_rep(const DecodeArgs& a, int rep, int n_seq, hipStream_t st) {
  switch (rep) {
    case 1: launch_t<DT, D, 1, FUSED>(a, n_seq, st); break;
    case 2: launch_t<DT, D, 2, FUSED>(a, n_seq, st); break;
    case 4: launch_t<DT, D, 4, FUSED>(a, n_seq, st); break;
    case 8: launch_t<DT, D, 8, FUSED>(a, n_seq, st); break;
    default: return fail(LNSKV_ERR_UNSUPPORTED, "n_heads/n_kv_heads = %d not supported (1, 2, 4, 8)", rep);
  }
  return hip_check("decode kernel launch");
}

template <int DT, bool FUSED>
int launch_decode_valu(const DecodeArgs& a, int d, int rep, int n_seq, hipStream_t st) {
  switch (d) {
    case 64: return launch_rep<DT, 64, FUSED>(a, rep, n_seq, st);
    case 128: return launch_rep<DT, 128, FUSED>(a, rep, n_seq, st);
    case 256: return launch_rep<DT, 256, FUSED>(a, rep, n_seq, st);
    default: return fail(LNSKV_ERR_UNSUPPORTED, "head_dim %d", d);
  }
}

template int launch_decode_valu<LNSKV_DTYPE_F32, false>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_valu<LNSKV_DTYPE_F32, true>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_valu<LNSKV_DTYPE_F16, false>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_valu<LNSKV_DTYPE_F16, true>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_valu<LNSKV_DTYPE_Q8A, false>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_valu<LNSKV_DTYPE_Q8A, true>(const DecodeArgs&, int, int, int, hipStream_t);

}  // namespace lnskv
