// Launchers of the matrix-core decode kernels (lnskv_decode_mfma.h) over the
// window [p_start, kv_len) of every sequence.
#include "lnskv_decode_mfma.h"

namespace lnskv {
namespace {
// RoPE variants exist for fused calls only (a.rope_half > 0).
template <int REP, bool FUSED, int NH>
void launch_mfma_rep(const DecodeArgs& a, int n_seq, hipStream_t st) {
  const dim3 grid((unsigned)a.n_kv, (unsigned)a.max_parts, (unsigned)n_seq);
  if (FUSED && a.rope_half > 0)
    decode_mfma_kernel<REP, FUSED, FUSED, NH><<<grid, kWave, 0, st>>>(a);
  else
    decode_mfma_kernel<REP, FUSED, false, NH><<<grid, kWave, 0, st>>>(a);
  launch_combine<REP, NH * kD, FUSED>(a, n_seq, st);
}

}  // namespace

template <bool FUSED>
int launch_decode_mfma_f16(const DecodeArgs& a, int rep, int d, int n_seq, hipStream_t st) {
  if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
        launch_mfma_rep<decltype(rep_c)::value, FUSED, decltype(nh_c)::value>(a, n_seq, st);
      }))
    return rc;
  return hip_check("decode kernel launch");
}

template int launch_decode_mfma_f16<false>(const DecodeArgs&, int, int, int, hipStream_t);
template int launch_decode_mfma_f16<true>(const DecodeArgs&, int, int, int, hipStream_t);

namespace {

// Resident waves of one stream-K kernel (ROPE: the fused variant that turns
// RoPE in registers, whose extra registers may fit fewer waves), capped at
// the launch shape's waves per CU.
template <int REP, bool FUSED, bool Q8, int NH, bool ROPE>
int sk_waves_of(int cus, int* waves) {
  int per_cu = 0;
  constexpr int depth = sk_depth<Q8, NH>();
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, decode_sk_kernel<REP, FUSED, depth, ROPE, Q8, NH>, kWave,
                                                   0) != hipSuccess)
    per_cu = 0;
  if (per_cu <= 0) return fail(LNSKV_ERR_HIP, "occupancy query of the stream-K decode kernel failed");
  *waves = cus * std::min(per_cu, Q8 ? kSkWavesPerCuQ8 : kSkWavesPerCu);
  return LNSKV_OK;
}

template <int REP, bool FUSED, int NH>
void launch_sk_rep(const DecodeArgs& a, int n_seq, int n_waves, bool q8, hipStream_t st) {
  const bool rope = FUSED && a.rope_half > 0;
  constexpr int dq = sk_depth<true, NH>(), df = sk_depth<false, NH>();
  if (q8 && rope)
    decode_sk_kernel<REP, FUSED, dq, FUSED, true, NH><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves);
  else if (q8)
    decode_sk_kernel<REP, FUSED, dq, false, true, NH><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves);
  else if (rope)
    decode_sk_kernel<REP, FUSED, df, FUSED, false, NH><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves);
  else
    decode_sk_kernel<REP, FUSED, df, false, false, NH><<<n_waves, kWave, 0, st>>>(a, n_seq, n_waves);
  combine_sk_kernel<REP, FUSED, NH><<<n_waves, kBlock, 0, st>>>(a, n_seq, n_waves);
}
}  // namespace

int mfma_sk_waves(int rep, int d, bool fused, bool q8, bool rope, int* waves) {
  // resident waves used per launch on the current device, kept per
  // (device, rep, head dim, fused, q8, rope)
  static std::mutex mu;
  static std::map<std::tuple<int, int, int, bool, bool, bool>, int> cache;
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(LNSKV_ERR_HIP, "hipGetDevice failed");
  rope = rope && fused;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(dev, rep, d, fused, q8, rope);
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
        auto of = [&](auto q8_c) {
          constexpr bool Q = decltype(q8_c)::value;
          if (!fused) return sk_waves_of<R, false, Q, NH, false>(cus, waves);
          return rope ? sk_waves_of<R, true, Q, NH, true>(cus, waves) : sk_waves_of<R, true, Q, NH, false>(cus, waves);
        };
        rc = q8 ? of(std::true_type{}) : of(std::false_type{});
      }))
    return r;
  if (rc == LNSKV_OK) cache[key] = *waves;
  return rc;
}

template <bool FUSED>
int launch_decode_mfma_sk(const DecodeArgs& a, int rep, int d, int n_seq, int n_waves, bool q8, hipStream_t st) {
  if (n_seq > kSkMaxSeqs)
    return fail(LNSKV_ERR_INVALID, "stream-K decode serves at most %d sequences", kSkMaxSeqs);
  if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
        launch_sk_rep<decltype(rep_c)::value, FUSED, decltype(nh_c)::value>(a, n_seq, n_waves, q8, st);
      }))
    return rc;
  return hip_check("stream-K decode kernel launch");
}

template int launch_decode_mfma_sk<false>(const DecodeArgs&, int, int, int, int, bool, hipStream_t);
template int launch_decode_mfma_sk<true>(const DecodeArgs&, int, int, int, int, bool, hipStream_t);

namespace {

template <int REP, bool FUSED, int NH>
void launch_wg_rep(const DecodeArgs& a, int n_seq, int n_wg, int n_cu, bool q8, hipStream_t st) {
  const bool rope = FUSED && a.rope_half > 0;
  if (q8 && rope)
    decode_wg_kernel<REP, FUSED, kSkDepthQ8, FUSED, true, kWgWavesQ8, NH>
        <<<n_wg, kWave * kWgWavesQ8, 0, st>>>(a, n_seq, n_wg, n_cu);
  else if (q8)
    decode_wg_kernel<REP, FUSED, kSkDepthQ8, false, true, kWgWavesQ8, NH>
        <<<n_wg, kWave * kWgWavesQ8, 0, st>>>(a, n_seq, n_wg, n_cu);
  else if (rope)
    decode_wg_kernel<REP, FUSED, kSkDepth, FUSED, false, kWgWaves, NH>
        <<<n_wg, kWave * kWgWaves, 0, st>>>(a, n_seq, n_wg, n_cu);
  else
    decode_wg_kernel<REP, FUSED, kSkDepth, false, false, kWgWaves, NH>
        <<<n_wg, kWave * kWgWaves, 0, st>>>(a, n_seq, n_wg, n_cu);
}
}  // namespace

int mfma_wg_count(int* n_wg) {
  // kWgPerCu workgroups per CU of the current device (at most kWgMaxGroups)
  static std::mutex mu;
  static std::map<int, int> cache;
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(LNSKV_ERR_HIP, "hipGetDevice failed");
  std::lock_guard<std::mutex> lock(mu);
  const auto it = cache.find(dev);
  if (it != cache.end()) {
    *n_wg = it->second;
    return LNSKV_OK;
  }
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    return fail(LNSKV_ERR_HIP, "compute-unit count query failed");
  const int n = std::min(cus * kWgPerCu, kWgMaxGroups);
  cache[dev] = n;
  *n_wg = n;
  return LNSKV_OK;
}

template <bool FUSED>
int launch_decode_mfma_wg(const DecodeArgs& a, int rep, int d, int n_seq, int n_wg, bool q8, hipStream_t st) {
  if (n_seq > kSkMaxSeqs)
    return fail(LNSKV_ERR_INVALID, "the workgroup schedule serves at most %d sequences", kSkMaxSeqs);
  if (n_wg <= 0 || n_wg > kWgMaxGroups) return fail(LNSKV_ERR_INVALID, "%d workgroups", n_wg);
  // Launch only the workgroups the batch can fill: with at most `bound`
  // units (from max_kv_len), groups of NW * kWgMinPages units each cover
  // them, so the kernel's chunk C = max(NW * kWgMinPages, ceil(T / G)) stays
  // at its minimum and [0, G * C) still holds every unit; one more per
  // segment lets the segment-aligned ranges (ceil(np / C) or fewer
  // workgroups per segment, at most T / C + n_seq n_kv in all) fit the grid.
  const int nw = q8 ? kWgWavesQ8 : kWgWaves;
  const int64_t bound = (int64_t)n_seq * a.n_kv * ((int64_t)a.max_kv_len / kPage + 1);
  const int64_t per = (int64_t)nw * kWgMinPages;
  const int n_cu = n_wg / kWgPerCu;
  int64_t want = (bound + per - 1) / per + (int64_t)n_seq * a.n_kv;
  if (!a.kv_len && !a.p_start) {
    // every sequence has the scalar window (the reference's one-sequence
    // call): exactly the kernel's segment-aligned count, np as in sk_fields
    int L = a.kv_len_scalar;
    L = L > std::min(a.max_kv_len, a.bt_stride * kPage) ? 0 : std::max(L, 0);
    const int p0 = std::min(std::max(a.p_start_scalar, 0), L);
    const int lo = FUSED && L > 0 ? std::min(p0, L - 1) : p0;
    const int64_t np = L > lo ? (L - 1) / kPage - lo / kPage + 1 : 0;
    const int64_t segs = (int64_t)n_seq * a.n_kv;
    want = segs * wg_seg_ceil((int)np, (int)per);
    if (want > n_cu) want = segs * (np > 0 ? std::max<int64_t>(1, np / per) : 0);
  }
  const int groups = (int)std::max<int64_t>(1, std::min<int64_t>(n_wg, want));
  if (int rc = with_rep_nh(rep, d, [&](auto rep_c, auto nh_c) {
        launch_wg_rep<decltype(rep_c)::value, FUSED, decltype(nh_c)::value>(a, n_seq, groups, n_cu, q8, st);
      }))
    return rc;
  return hip_check("workgroup decode kernel launch");
}

template int launch_decode_mfma_wg<false>(const DecodeArgs&, int, int, int, int, bool, hipStream_t);
template int launch_decode_mfma_wg<true>(const DecodeArgs&, int, int, int, int, bool, hipStream_t);

}  // namespace lnskv
