// Decode with a sliding window whose first tokens stay visible: query row s
// attends tokens t < n_sink and t >= kv_len - window of its sequence.
//
// The decode kernels' kSink variant: a sequence's pages are counted without the
// gap between the sinks' pages and the window's (one compare and add per table
// entry), so that every schedule divides exactly the pages that are read; a
// page that holds both attended and other tokens is masked token by token.
// Bound by HBM like the plain decode: sinks + window tokens of K and V.  32 sequences of
// 512 to 16384 tokens, 32 heads on 8 of f16, window 4096 + 4: 96 us (stream-K; 480 MB at a
// large copy's 4.8 TB/s take 100).  One sequence of 32768, Q8A, window 1024 + 4: 13.7 us,
// the latency of table, pages and one merge between workgroups.
#include "lnskv_decode_block.h"
#include "lnskv_decode_var.h"

namespace lnskv {
namespace {

constexpr int kMaxSink = 1 << 30;
// Pages of a sequence up to which one workgroup per (sequence, kv head) takes them all,
// and up to which it does where those workgroups are about as many as compute units.
// Us, that | the plain decode's schedules: 17 sequences x 4 kv heads, window 84 + 61, Q8A
// 9.4 | 15.6; 16 x 4, 281 + 61, f16 8.9 | 12.9; 1 x 8, 102 + 55, f16 7.8 | 11.7; 18 x 4
// 256-wide, 182 + 58, Q8A 16.7 | 18.1; 60 x 4, 854 + 4, Q8A 18.4 | 23.2; but 6 x 4, 873 +
// 39, Q8A 19.0 | 12.2 and 1 x 8, 1024 + 4, Q8A 20.3 | 13.7.
constexpr int kBlockPages = 32;
constexpr int kBlockPagesFull = 64;

// A workgroup per (sequence, kv head): bound by the latency of its four waves' chains
// of at most 16 pages each.
template <int REP, bool Q8, int NH>
__global__ __launch_bounds__(kWave* kBlockWaves) __attribute__((amdgpu_waves_per_eu(NH == 1 ? 2 : 1)))
void sink_block_kernel(DecodeArgs a, VarArgs<kSink> x) {
  constexpr int NW = kBlockWaves, D = NH * kD, C = D / kWave;
  __shared__ BlockLds<REP, Q8, NH> sm;
  const int wi = (int)(threadIdx.x / kWave), lane = (int)(threadIdx.x % kWave);
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv), s = (int)(blockIdx.x / (unsigned)a.n_kv);
  int L = a.kv_len[s];
  L = L > min(a.max_kv_len, a.bt_stride * kPage) ? 0 : max(L, 0);
  const SinkSpan sp = sink_span(x, L);
  const int np = L > 0 ? (L - 1) / kPage + 1 - sp.gap : 0;
  const int per = (np + NW - 1) / NW, i0 = min(np, wi * per), i1 = min(np, i0 + per);
  if (i0 < i1) {
    PieceLoads<REP, NH> pl;
    piece_loads<REP, false, false, Q8, NH, kSink>(a, s, kvh, i0, pl, sp);
    block_piece<REP, Q8, NH, kSink>(a, sm, wi, s, kvh, pl, 0, i0, i1, L, sp);
  }
  __syncthreads();
  const int nw = np > 0 ? (np + per - 1) / per : 0;  // waves that left rows
  for (int h = wi; h < REP; h += NW) {  // wave-uniform
    float M, Ls, A[C];
    block_merge<REP, Q8, NH>(sm, nw, h, M, Ls, A);
    const size_t row = ((size_t)s * a.n_heads + (size_t)kvh * REP + h) * D;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const size_t i = row + c * kWave + lane;
      a.out[i] = gated(a, i, Ls > 0.0f ? A[c] / Ls : 0.0f);
    }
  }
}

int64_t sink_pages(int max_kv_len, int window, int n_sink) {
  const int64_t all = (int64_t)max_kv_len / kPage + 1;
  if (window <= 0) return all;
  return std::min(all, ((int64_t)window + kPage - 2) / kPage + 1 + ((int64_t)n_sink + kPage - 1) / kPage);
}

template <int REP, int NH, bool Q8>
int sink_waves_of(int cus, int* waves) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &per_cu, decode_sk_kernel<REP, false, sk_depth<Q8, NH>(), false, Q8, NH, kSink, VarArgs<kSink>>, kWave, 0) != hipSuccess)
    per_cu = 0;
  if (per_cu <= 0) return fail(LNSKV_ERR_HIP, "occupancy query of the stream-K decode kernel failed");
  *waves = cus * std::min(per_cu, Q8 ? kSkWavesPerCuQ8 : kSkWavesPerCu);
  return LNSKV_OK;
}

// Resident waves of the stream-K kernel on the current device, kept per
// (device, rep, head dim, Q8A).
int sink_sk_waves(int rep, int d, bool q8, int* waves) {
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
        rc = q8 ? sink_waves_of<R, NH, true>(cus, waves) : sink_waves_of<R, NH, false>(cus, waves);
      }))
    return r;
  if (rc == LNSKV_OK) cache[key] = *waves;
  return rc;
}

// units: the batch's (sequence, kv head, page) units at most; pages: a sequence's.
int plan_sink(const lnskv_pages* c, int n_seq, int n_heads, int64_t units, int64_t pages, VarPlan* p) {
  const int n_kv = (int)c->n_kv_heads, d = (int)c->head_dim, rep = n_heads / n_kv;
  *p = VarPlan{};
  if (!var_mfma(c)) return plan_tiles(c, n_seq, n_heads, pages, p);
  const int setting = schedule_setting();
  if (setting == kScheduleAuto && pages <= ((int64_t)n_seq * n_kv >= 192 ? kBlockPagesFull : kBlockPages)) {
    p->block = true;
    return LNSKV_OK;
  }
  // the workgroup schedule or stream-K by the size of the batch, as the plain decode
  if (units >= ((int64_t)1 << 30)) return fail(LNSKV_ERR_UNSUPPORTED, "a batch of more than 2^30 page units");
  int n_wg = 0;
  if (int rc = mfma_wg_count(&n_wg)) return rc;
  if (n_seq <= kSkMaxSeqs &&
      (setting == kScheduleWorkgroup || (setting == kScheduleAuto && units <= (int64_t)kWgSmallPages * n_wg))) {
    p->wg = n_wg;
    p->ws_bytes = kWsHeaderBytes + (size_t)n_wg * 2 * rep * ((size_t)d + 2) * sizeof(float);
    return LNSKV_OK;
  }
  if (int rc = sink_sk_waves(rep, d, c->dtype == LNSKV_DTYPE_Q8A, &p->sk_waves)) return rc;
  p->ws_bytes = kWsHeaderBytes + (size_t)p->sk_waves * (2 * rep * ((size_t)d + 2) * sizeof(float) + 16);
  return LNSKV_OK;
}

template <int REP, int NH>
void launch_sink_wg(const DecodeArgs& a, const VarArgs<kSink>& x, int n_seq, int n_wg, int n_cu, bool q8, hipStream_t st) {
  if (q8)
    decode_wg_kernel<REP, false, kSkDepthQ8, false, true, kWgWavesQ8, NH, kSink>
        <<<n_wg, kWave * kWgWavesQ8, 0, st>>>(a, n_seq, n_wg, n_cu, x);
  else
    decode_wg_kernel<REP, false, kSkDepth, false, false, kWgWaves, NH, kSink>
        <<<n_wg, kWave * kWgWaves, 0, st>>>(a, n_seq, n_wg, n_cu, x);
}

template <int REP, int NH>
void launch_sink_sk(const DecodeArgs& a, const VarArgs<kSink>& x, int n_seq, int n_waves, bool q8, hipStream_t st) {
  if (q8)
    decode_sk_kernel<REP, false, sk_depth<true, NH>(), false, true, NH, kSink><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves, x);
  else
    decode_sk_kernel<REP, false, sk_depth<false, NH>(), false, false, NH, kSink><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves, x);
  combine_sk_kernel<REP, false, NH, kSink><<<n_waves, kBlock, 0, st>>>(a, n_seq, n_waves, x);
}

// Launches the plan; ws: plan.ws_bytes of workspace.
int launch_plan(const lnskv_pages* c, DecodeArgs a, const VarPlan& plan, int64_t units, int n_seq, void* ws,
                const VarArgs<kSink>& x, hipStream_t st) {
  const int d = (int)c->head_dim, rep = a.n_heads / a.n_kv;
  const bool q8 = c->dtype == LNSKV_DTYPE_Q8A;
  uint8_t* body = static_cast<uint8_t*>(ws) + (ws ? kWsHeaderBytes : 0);
  if (plan.block) {
    const unsigned blocks = (unsigned)(n_seq * a.n_kv);
    if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
          constexpr int R = decltype(rep_c)::value, NH = decltype(nh_c)::value;
          if (q8) sink_block_kernel<R, true, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x);
          else sink_block_kernel<R, false, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x);
        }))
      return rc;
    return hip_check("decode kernel launch");
  }
  if (plan.wg > 0) {
    a.wg_cnt = static_cast<uint32_t*>(ws);
    a.ws_acc = reinterpret_cast<float*>(body);
    a.ws_ml = a.ws_acc + (size_t)plan.wg * 2 * rep * d;
    // as many workgroups as the batch can fill (launch_decode_mfma_wg)
    const int64_t per = (int64_t)(q8 ? kWgWavesQ8 : kWgWaves) * kWgMinPages;
    const int64_t want = (units + per - 1) / per + (int64_t)n_seq * a.n_kv;
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(plan.wg, want));
    if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
          launch_sink_wg<decltype(rep_c)::value, decltype(nh_c)::value>(a, x, n_seq, groups,
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
            launch_sink_sk<decltype(rep_c)::value, decltype(nh_c)::value>(
                b, x, std::min(n_seq - s0, kSkMaxSeqs), n_waves, q8, st);
          }))
        return rc;
      if (int rc = hip_check("stream-K decode kernel launch")) return rc;
    }
    return LNSKV_OK;
  }
  return launch_tiles<kSink>(c, a, plan, n_seq, ws, x, st);
}

int check_sink(int window, int n_sink) {
  if (window < 0) return fail(LNSKV_ERR_INVALID, "window %d is negative", window);
  if (n_sink < 0 || n_sink > kMaxSink) return fail(LNSKV_ERR_INVALID, "n_sink %d out of range [0, 2^30]", n_sink);
  return LNSKV_OK;
}

}  // namespace
}  // namespace lnskv

using namespace lnskv;

extern "C" {

int lnskv_sink_decode_workspace_size(const lnskv_pages* c, int32_t n_seq, int32_t n_heads, int32_t max_kv_len,
                                     int32_t window, int32_t n_sink, size_t* bytes) {
  clear_error();
  if (!bytes) return fail(LNSKV_ERR_INVALID, "bytes is NULL");
  *bytes = 0;
  if (int rc = check_geometry(c)) return rc;
  if (int rc = check_var_shape(c, n_seq, n_heads, max_kv_len)) return rc;
  if (int rc = check_sink(window, n_sink)) return rc;
  const int64_t pages = sink_pages(max_kv_len, window, n_sink);
  VarPlan plan;
  if (int rc = plan_sink(c, n_seq, n_heads, pages * n_seq * c->n_kv_heads, pages, &plan)) return rc;
  *bytes = plan.ws_bytes;
  return LNSKV_OK;
}

int lnskv_sink_decode(const lnskv_pages* c, const float* q, float* out, const float* gate, const uint32_t* bt,
                      int32_t bt_stride, const int32_t* kv_len, int32_t n_seq, int32_t n_heads, int32_t max_kv_len,
                      int32_t window, int32_t n_sink, float scale, void* ws, size_t ws_bytes, lnskv_stream_t stream) {
  clear_error();
  if (int rc = check_var_call(c, q, out, bt, bt_stride, kv_len, n_seq, n_heads, max_kv_len, scale)) return rc;
  if (int rc = check_var_shape(c, n_seq, n_heads, max_kv_len)) return rc;
  if (int rc = check_sink(window, n_sink)) return rc;
  const int64_t pages = sink_pages(max_kv_len, window, n_sink), units = pages * n_seq * c->n_kv_heads;
  VarPlan plan;
  if (int rc = plan_sink(c, n_seq, n_heads, units, pages, &plan)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = var_workspace(&ws, ws_bytes, plan.ws_bytes, st)) return rc;
  const DecodeArgs a = var_args(c, q, out, gate, bt, bt_stride, kv_len, n_heads, max_kv_len, scale, plan, stream);
  return launch_plan(c, a, plan, units, n_seq, ws, VarArgs<kSink>{window, n_sink}, st);
}

}  // extern "C"
