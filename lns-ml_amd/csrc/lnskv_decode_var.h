// Host side of the decode variants (kSink, kPrefix): the plan of a call and
// the launches of the matrix-core and generic decode kernels with VarArgs.
#pragma once

#include <cmath>

#include "lnskv_decode_mfma.h"
#include "lnskv_decode_valu.h"

namespace lnskv {
namespace {

// How a call runs: on f16 and Q8A pages with head_dim 128 or 256 the workgroup
// schedule (wg > 0) or stream-K (sk_waves > 0) by the size of the batch, as
// the plain decode, in launches of at most kSkMaxSeqs sequences; on other
// pages the generic kernel in partitions of `split` tokens.
struct VarPlan {
  int wg = 0;
  int sk_waves = 0;
  int split = 0;
  int max_parts = 1;
  size_t ws_bytes = 0;
};

inline bool var_mfma(const lnskv_pages* c) {
  return c->dtype != LNSKV_DTYPE_F32 && (c->head_dim == 128 || c->head_dim == 256);
}

template <int VAR, int REP, int NH, bool Q8>
int var_waves_of(int cus, int* waves) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &per_cu, decode_sk_kernel<REP, false, sk_depth<Q8, NH>(), false, Q8, NH, VAR, VarArgs<VAR>>, kWave, 0) != hipSuccess)
    per_cu = 0;
  if (per_cu <= 0) return fail(LNSKV_ERR_HIP, "occupancy query of the stream-K decode kernel failed");
  *waves = cus * std::min(per_cu, Q8 ? kSkWavesPerCuQ8 : kSkWavesPerCu);
  return LNSKV_OK;
}

// Resident waves of the stream-K kernel on the current device, kept per
// (device, rep, head dim, Q8A).
template <int VAR>
int var_sk_waves(int rep, int d, bool q8, int* waves) {
  static std::mutex mu;
  static std::map<std::tuple<int, int, int, bool>, int> cache;
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(LNSKV_ERR_HIP, "hipGetDevice failed");
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(dev, rep, d, q8);
  const auto it = cache.find(key);
  if (it != cache.end()) {
    *waves = it->second;
    return LNSKV_OK;
  }
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    return fail(LNSKV_ERR_HIP, "compute-unit count query failed");
  int rc = LNSKV_OK;
  if (int r = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
        constexpr int R = decltype(rep_c)::value, NH = decltype(nh_c)::value;
        rc = q8 ? var_waves_of<VAR, R, NH, true>(cus, waves) : var_waves_of<VAR, R, NH, false>(cus, waves);
      }))
    return r;
  if (rc == LNSKV_OK) cache[key] = *waves;
  return rc;
}

// units: the batch's (sequence, kv head, page) units at most; max_pages: a
// sequence's pages at most; from_zero: which start at position 0 (partitions
// of the generic kernel start at multiples of `split`, so that others may touch
// one more).
template <int VAR>
int plan_var(const lnskv_pages* c, int n_seq, int n_heads, int64_t units, int64_t max_pages, bool from_zero,
             VarPlan* p) {
  const int n_kv = (int)c->n_kv_heads, d = (int)c->head_dim, rep = n_heads / n_kv;
  *p = VarPlan{};
  if (var_mfma(c)) {
    if (units >= ((int64_t)1 << 30)) return fail(LNSKV_ERR_UNSUPPORTED, "a batch of more than 2^30 page units");
    int n_wg = 0;
    if (int rc = mfma_wg_count(&n_wg)) return rc;
    const int setting = schedule_setting();
    if (n_seq <= kSkMaxSeqs &&
        (setting == kScheduleWorkgroup || (setting == kScheduleAuto && units <= (int64_t)kWgSmallPages * n_wg))) {
      p->wg = n_wg;
      p->ws_bytes = kWsHeaderBytes + (size_t)n_wg * 2 * rep * ((size_t)d + 2) * sizeof(float);
      return LNSKV_OK;
    }
    if (int rc = var_sk_waves<VAR>(rep, d, c->dtype == LNSKV_DTYPE_Q8A, &p->sk_waves)) return rc;
    p->ws_bytes = kWsHeaderBytes + (size_t)p->sk_waves * (2 * rep * ((size_t)d + 2) * sizeof(float) + 16);
    return LNSKV_OK;
  }
  const int64_t tokens = max_pages * kPage;
  p->split = choose_split(n_seq, n_kv, (int)std::min<int64_t>(tokens, INT32_MAX / 2));
  const int64_t parts = std::max<int64_t>(1, (tokens + p->split - 1) / p->split + (from_zero ? 0 : 1));
  if (parts > 65535) return fail(LNSKV_ERR_INVALID, "%lld tokens a sequence need more than 65535 partitions", (long long)tokens);
  p->max_parts = (int)parts;
  p->ws_bytes =
      parts > 1 ? kWsHeaderBytes + (size_t)n_seq * n_heads * parts * ((size_t)d + 2) * sizeof(float) : 0;
  return LNSKV_OK;
}

template <int VAR, int REP, int NH>
void launch_var_wg(const DecodeArgs& a, const VarArgs<VAR>& x, int n_seq, int n_wg, int n_cu, bool q8, hipStream_t st) {
  if (q8)
    decode_wg_kernel<REP, false, kSkDepthQ8, false, true, kWgWavesQ8, NH, VAR>
        <<<n_wg, kWave * kWgWavesQ8, 0, st>>>(a, n_seq, n_wg, n_cu, x);
  else
    decode_wg_kernel<REP, false, kSkDepth, false, false, kWgWaves, NH, VAR>
        <<<n_wg, kWave * kWgWaves, 0, st>>>(a, n_seq, n_wg, n_cu, x);
}

template <int VAR, int REP, int NH>
void launch_var_sk(const DecodeArgs& a, const VarArgs<VAR>& x, int n_seq, int n_waves, bool q8, hipStream_t st) {
  if (q8)
    decode_sk_kernel<REP, false, sk_depth<true, NH>(), false, true, NH, VAR><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves, x);
  else
    decode_sk_kernel<REP, false, sk_depth<false, NH>(), false, false, NH, VAR><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves, x);
  combine_sk_kernel<REP, false, NH, VAR><<<n_waves, kBlock, 0, st>>>(a, n_seq, n_waves, x);
}

template <int VAR, int DT, int D, int REP>
void launch_var_valu(const DecodeArgs& a, const VarArgs<VAR>& x, int n_seq, hipStream_t st) {
  const dim3 grid((unsigned)a.n_kv, (unsigned)a.max_parts, (unsigned)n_seq);
  decode_valu_kernel<DT, D, REP, false, VAR><<<grid, kBlock, 0, st>>>(a, x);
  launch_combine<REP, D, false, VAR>(a, n_seq, st, x);
}

template <int VAR, int DT, int D>
int launch_var_valu_rep(const DecodeArgs& a, const VarArgs<VAR>& x, int rep, int n_seq, hipStream_t st) {
  switch (rep) {
    case 1: launch_var_valu<VAR, DT, D, 1>(a, x, n_seq, st); break;
    case 2: launch_var_valu<VAR, DT, D, 2>(a, x, n_seq, st); break;
    case 4: launch_var_valu<VAR, DT, D, 4>(a, x, n_seq, st); break;
    default: launch_var_valu<VAR, DT, D, 8>(a, x, n_seq, st); break;
  }
  return hip_check("decode kernel launch");
}

// The arguments every variant checks alike.
inline int check_var_call(const lnskv_pages* c, const float* q, const float* out, const uint32_t* bt, int bt_stride,
                          const int32_t* kv_len, int n_seq, int n_heads, int max_kv_len, float scale) {
  if (int rc = check_pages(c)) return rc;
  if (!q || !out || !bt || !kv_len) return fail(LNSKV_ERR_INVALID, "q, out, block tables and kv_len must be non-null");
  if (bt_stride <= 0) return fail(LNSKV_ERR_INVALID, "bt_stride %d must be positive", bt_stride);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(LNSKV_ERR_INVALID, "scale must be positive and finite");
  return LNSKV_OK;
}
inline int check_var_shape(const lnskv_pages* c, int n_seq, int n_heads, int max_kv_len) {
  if (n_seq <= 0 || n_seq > 65535) return fail(LNSKV_ERR_INVALID, "n_seq %d out of range [1, 65535]", n_seq);
  if (n_heads <= 0 || n_heads % (int)c->n_kv_heads != 0)
    return fail(LNSKV_ERR_INVALID, "n_heads %d is not a multiple of n_kv_heads %u", n_heads, c->n_kv_heads);
  const int rep = n_heads / (int)c->n_kv_heads;
  if (rep != 1 && rep != 2 && rep != 4 && rep != 8)
    return fail(LNSKV_ERR_UNSUPPORTED, "n_heads/n_kv_heads = %d not supported (1, 2, 4, 8)", rep);
  if (max_kv_len < 0) return fail(LNSKV_ERR_INVALID, "max_kv_len %d is negative", max_kv_len);
  return LNSKV_OK;
}

inline DecodeArgs var_args(const lnskv_pages* c, const float* q, float* out, const float* gate, const uint32_t* bt,
                           int bt_stride, const int32_t* kv_len, int n_heads, int max_kv_len, float scale,
                           const VarPlan& plan, lnskv_stream_t stream) {
  DecodeArgs a{};
  a.k_pages = static_cast<const uint8_t*>(c->k_pages);
  a.v_pages = static_cast<const uint8_t*>(c->v_pages);
  a.k_scales = c->k_scales;
  a.v_scales = c->v_scales;
  a.q = q;
  a.out = out;
  a.gate = gate;
  a.bt = bt;
  a.bt_stride = bt_stride;
  a.kv_len = kv_len;
  a.n_kv = (int32_t)c->n_kv_heads;
  a.n_heads = n_heads;
  a.split = plan.split;
  a.max_parts = plan.max_parts;
  a.max_kv_len = max_kv_len;
  a.num_pages = c->num_pages;
  a.scale_log2 = scale * kLog2e;
  a.ws_err = ws_error_word(stream, true);
  return a;
}

// Launches the plan; ws: plan.ws_bytes of workspace.  seq_args(s0): the
// variant's arguments of a launch that starts at sequence s0.
template <int VAR, class F>
int launch_plan(const lnskv_pages* c, DecodeArgs a, const VarPlan& plan, int64_t units, int n_seq, void* ws,
                hipStream_t st, F&& seq_args) {
  const int d = (int)c->head_dim, rep = a.n_heads / a.n_kv;
  const bool q8 = c->dtype == LNSKV_DTYPE_Q8A;
  uint8_t* body = static_cast<uint8_t*>(ws) + (ws ? kWsHeaderBytes : 0);
  if (plan.wg > 0) {
    a.wg_cnt = static_cast<uint32_t*>(ws);
    a.ws_acc = reinterpret_cast<float*>(body);
    a.ws_ml = a.ws_acc + (size_t)plan.wg * 2 * rep * d;
    // as many workgroups as the batch can fill (launch_decode_mfma_wg)
    const int64_t per = (int64_t)(q8 ? kWgWavesQ8 : kWgWaves) * kWgMinPages;
    const int64_t want = (units + per - 1) / per + (int64_t)n_seq * a.n_kv;
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(plan.wg, want));
    if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
          launch_var_wg<VAR, decltype(rep_c)::value, decltype(nh_c)::value>(a, seq_args(0), n_seq, groups,
                                                                             plan.wg / kWgPerCu, q8, st);
        }))
      return rc;
    return hip_check("workgroup decode kernel launch");
  }
  if (plan.sk_waves > 0) {
    const int n_waves = plan.sk_waves;
    a.ws_acc = reinterpret_cast<float*>(body);
    a.ws_ml = a.ws_acc + (size_t)n_waves * 2 * rep * d;
    a.sk_desc = reinterpret_cast<int4*>(a.ws_ml + (size_t)n_waves * 2 * rep * 2);
    for (int s0 = 0; s0 < n_seq; s0 += kSkMaxSeqs) {  // the launches share the workspace in stream order
      DecodeArgs b = a;
      const size_t qo = (size_t)s0 * a.n_heads * d;
      b.q = a.q + qo;
      b.out = a.out + qo;
      b.gate = a.gate ? a.gate + qo : nullptr;
      b.bt = a.bt + (size_t)s0 * a.bt_stride;
      b.kv_len = a.kv_len + s0;
      if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
            launch_var_sk<VAR, decltype(rep_c)::value, decltype(nh_c)::value>(
                b, seq_args(s0), std::min(n_seq - s0, kSkMaxSeqs), n_waves, q8, st);
          }))
        return rc;
      if (int rc = hip_check("stream-K decode kernel launch")) return rc;
    }
    return LNSKV_OK;
  }
  if (plan.ws_bytes > 0) {
    a.ws_acc = reinterpret_cast<float*>(body);
    a.ws_ml = a.ws_acc + (size_t)n_seq * a.n_heads * plan.max_parts * d;
  }
  const VarArgs<VAR> x = seq_args(0);
  if (c->dtype == LNSKV_DTYPE_F32) {
    switch (d) {
      case 64: return launch_var_valu_rep<VAR, LNSKV_DTYPE_F32, 64>(a, x, rep, n_seq, st);
      case 128: return launch_var_valu_rep<VAR, LNSKV_DTYPE_F32, 128>(a, x, rep, n_seq, st);
      default: return launch_var_valu_rep<VAR, LNSKV_DTYPE_F32, 256>(a, x, rep, n_seq, st);
    }
  }
  if (q8) return launch_var_valu_rep<VAR, LNSKV_DTYPE_Q8A, 64>(a, x, rep, n_seq, st);
  return launch_var_valu_rep<VAR, LNSKV_DTYPE_F16, 64>(a, x, rep, n_seq, st);
}

// A call's workspace: the caller's, checked, or the library's decode buffer.
inline int var_workspace(void** ws, size_t ws_bytes, size_t need, hipStream_t st) {
  if (*ws == nullptr) return need > 0 ? library_buffer(0, need, ws, st) : LNSKV_OK;
  if (reinterpret_cast<uintptr_t>(*ws) % 16 != 0)
    return fail(LNSKV_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  if (ws_bytes < need) return fail(LNSKV_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, need);
  return LNSKV_OK;
}

}  // namespace
}  // namespace lnskv
