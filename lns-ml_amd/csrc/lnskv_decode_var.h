// Host side shared by the decode variants (kSink, kPrefix): the checks of a
// call, its arguments and workspace, and the tile kernel's launches.
#pragma once

#include <cmath>

#include <algorithm>

#include "lnskv_decode_tile.h"

namespace lnskv {
namespace {

// How a call runs.  On f16 and Q8A pages with head_dim 128 or 256 (var_mfma) each
// variant has schedules of its own; on other pages the tile kernel runs in
// partitions of `split` tokens.
struct VarPlan {
  bool block = false;  // kSink: a workgroup per (sequence, kv head)
  int wg = 0;          // kSink: the workgroup schedule
  int sk_waves = 0;    // kSink: stream-K
  int split = 0;
  int max_parts = 1;
  size_t ws_bytes = 0;
};

// Tokens of a sequence up to which one block takes them all, and the fewest that a
// partition has otherwise (a second launch merges partitions).  kOnePartitionFull where the
// (sequence, kv head) pairs are about as many as the compute units, else by what a page's
// products cost.  Us, one block | partitions, 12 sequences x 4 kv heads of 8 heads: f16
// 64-wide, 352 tokens 7.7 | 9.4, 480 8.5 | 9.9, 560 9.1 | 9.0; Q8A 352 9.0 | 9.7, 480 10.4 |
// 9.6; f32 288 8.8 | 9.4, 352 10.0 | 9.5, 416 11.3 | 9.6; f32 128-wide, 2 x 8 of 288 11.7 |
// 10.9, of 352 13.5 | 10.9; full, 48 x 4 of 700, f32 16.8 | 21.5, f32 256-wide 54.7 | 84.0,
// f16 in f32 products 18.7 | 19.2, of 960 23.3 | 21.8.  Partitions of 64 | 128 | 192 | 256 |
// 512 tokens: 24 x 4 of 1021, f32 16.6 | 15.3 | 17.5 | 15.8 | 19.5; 3 x 4 of 3700, Q8A 12.3 |
// 11.0 | 10.9 | 11.6 | 16.2.
constexpr int kOnePartitionFull = 768;
constexpr int kLeastPartition = 128;
inline int one_partition(const lnskv_pages* c, int n_seq) {
  if ((int64_t)n_seq * c->n_kv_heads >= 192) return kOnePartitionFull;
  return c->head_dim > 64 ? 256 : c->dtype == LNSKV_DTYPE_F16 ? 512 : 352;
}

inline bool var_mfma(const lnskv_pages* c) {
  return c->dtype != LNSKV_DTYPE_F32 && (c->head_dim == 128 || c->head_dim == 256);
}

// The tile kernel's partitions for sequences of at most `pages` pages: one
// where those are few (a block's four waves share it and no merge is launched).
inline int plan_tiles(const lnskv_pages* c, int n_seq, int n_heads, int64_t pages, VarPlan* p) {
  const int64_t tokens = std::max<int64_t>(pages, 1) * kPage;
  p->split = (int)tokens;
  if (tokens > one_partition(c, n_seq))
    p->split = std::max(kLeastPartition, choose_split(n_seq, (int)c->n_kv_heads, (int)std::min<int64_t>(tokens, INT32_MAX / 2)));
  const int64_t parts = (tokens + p->split - 1) / p->split;
  if (parts > 65535)
    return fail(LNSKV_ERR_INVALID, "%lld tokens a sequence need more than 65535 partitions", (long long)tokens);
  p->max_parts = (int)parts;
  p->ws_bytes = parts > 1 ? kWsHeaderBytes + (size_t)n_seq * n_heads * parts * ((size_t)c->head_dim + 2) * sizeof(float) : 0;
  return LNSKV_OK;
}

template <int VAR, int DT, int D, int REP>
void launch_tile(const DecodeArgs& a, const VarArgs<VAR>& x, int n_seq, hipStream_t st) {
  const dim3 grid((unsigned)a.n_kv, (unsigned)a.max_parts, (unsigned)n_seq);
  decode_tile_kernel<DT, D, REP, VAR><<<grid, kBlock, 0, st>>>(a, x);
  launch_combine<REP, D, false, VAR>(a, n_seq, st, x);
}

template <int VAR, int DT, int D>
int launch_tile_rep(const DecodeArgs& a, const VarArgs<VAR>& x, int rep, int n_seq, hipStream_t st) {
  switch (rep) {
    case 1: launch_tile<VAR, DT, D, 1>(a, x, n_seq, st); break;
    case 2: launch_tile<VAR, DT, D, 2>(a, x, n_seq, st); break;
    case 4: launch_tile<VAR, DT, D, 4>(a, x, n_seq, st); break;
    default: launch_tile<VAR, DT, D, 8>(a, x, n_seq, st); break;
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

// Launches the tile kernel; ws: plan.ws_bytes of workspace.
template <int VAR>
int launch_tiles(const lnskv_pages* c, DecodeArgs a, const VarPlan& plan, int n_seq, void* ws, const VarArgs<VAR>& x,
                   hipStream_t st) {
  const int d = (int)c->head_dim, rep = a.n_heads / a.n_kv;
  if (plan.ws_bytes > 0) {
    a.ws_acc = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kWsHeaderBytes);
    a.ws_ml = a.ws_acc + (size_t)n_seq * a.n_heads * plan.max_parts * d;
  }
  if (c->dtype == LNSKV_DTYPE_F32) {
    switch (d) {
      case 64: return launch_tile_rep<VAR, LNSKV_DTYPE_F32, 64>(a, x, rep, n_seq, st);
      case 128: return launch_tile_rep<VAR, LNSKV_DTYPE_F32, 128>(a, x, rep, n_seq, st);
      default: return launch_tile_rep<VAR, LNSKV_DTYPE_F32, 256>(a, x, rep, n_seq, st);
    }
  }
  if (c->dtype == LNSKV_DTYPE_Q8A) return launch_tile_rep<VAR, LNSKV_DTYPE_Q8A, 64>(a, x, rep, n_seq, st);
  return launch_tile_rep<VAR, LNSKV_DTYPE_F16, 64>(a, x, rep, n_seq, st);
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
