// Decode with a sliding window whose first tokens stay visible: query row s
// attends tokens t < n_sink and t >= kv_len - window of its sequence.
//
// The decode kernels' kSink variant: a sequence's pages are counted without the
// gap between the sinks' pages and the window's (one compare and add per table
// entry), so that every schedule divides exactly the pages that are read; a
// page that holds both attended and other tokens is masked token by token.
// Bound by HBM like the plain decode: sinks + window tokens of K and V.
#include "lnskv_decode_var.h"

namespace lnskv {
namespace {

constexpr int kMaxSink = 1 << 30;

int64_t sink_pages(int max_kv_len, int window, int n_sink) {
  const int64_t all = (int64_t)max_kv_len / kPage + 1;
  if (window <= 0) return all;
  return std::min(all, ((int64_t)window + kPage - 2) / kPage + 1 + ((int64_t)n_sink + kPage - 1) / kPage);
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
  if (int rc = plan_var<kSink>(c, n_seq, n_heads, pages * n_seq * c->n_kv_heads, pages, true, &plan)) return rc;
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
  if (int rc = plan_var<kSink>(c, n_seq, n_heads, units, pages, true, &plan)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = var_workspace(&ws, ws_bytes, plan.ws_bytes, st)) return rc;
  const DecodeArgs a = var_args(c, q, out, gate, bt, bt_stride, kv_len, n_heads, max_kv_len, scale, plan, stream);
  return launch_plan<kSink>(c, a, plan, units, n_seq, ws, st, [&](int) { return VarArgs<kSink>{window, n_sink}; });
}

}  // extern "C"
