// Append with rotary positions of several axes: q and the new K turned by the
// positions of up to four axes (time, height, width, ...), K and V converted
// to the page type and stored, in one pass over the rows.
//
// Pair i (dims i and i + half of a head, i < half = rotary_dim / 2) belongs to
// one axis a(i); token t turns it by angle pos[a(i)][t] * inv_freqs[i]:
//   y_i = x_i cos - x_{i+half} sin,  y_{i+half} = x_i sin + x_{i+half} cos
// The angle is the f64 product and its sine and cosine an f64 evaluation
// rounded once to f32, so far positions lose nothing (an f32 product is off by
// up to 2^-25 of the angle: 4e-3 rad at position 131072); products and sums of
// the turn are f32, each rounded once.
//
// A row is one head of one token.  D/8 lanes hold it, eight elements each: the
// lanes of the turned part the four dims 4l .. and their partners half + 4l ..,
// so that the turn needs no exchange, the others eight dims in a row; loads and
// stores are 16 bytes per lane either way.  A block takes one token (or a share of
// its rows): its first `half` threads make the token's (sin, cos) table in LDS
// once for every head while the first rows are on their way from memory.
//
// Bound by HBM: q read and written in f32, K and V read in f32 and written in
// the page type.  4096 tokens of 16 q and 2 x 4 K and V heads of 256, Q8A pages: 35.5 us
// (176 MB, 4.9 TB/s; a large copy reaches 4.8).  32 tokens of 32 q and 2 x 8 heads of
// 128: 3.0 us, a launch.  1001 tokens of 64-wide f32 heads with 44 dims turned (22 pairs,
// loads of one element): 8.8 us, 4.3 at the copy's rate.
#include <cmath>

#include "lnskv_device.h"

namespace lnskv {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxHalf = 128;  // head_dim 256

struct MropeArgs {
  uint8_t* k_pages;
  uint8_t* v_pages;
  float* k_scales;
  float* v_scales;
  const float* q;  // nullptr: no queries (n_heads 0)
  float* q_out;
  const float* k_new;
  const float* v_new;
  const int32_t* axis_pos;  // [n_axes][n_tok]
  const int32_t* tok_seq;
  const int32_t* tok_pos;
  const uint32_t* bt;
  const float* inv;
  int32_t sec[kMaxAxes];  // pairs of each axis
  int32_t n_axes;
  int32_t interleaved;
  int32_t half;
  int32_t n_tok;
  int32_t n_heads;
  int32_t n_kv;
  int32_t n_rows;
  int32_t bt_stride;
  int32_t rows_per_block;
  uint32_t num_pages;
};

// The axis that turns pair i.
__device__ __forceinline__ int pair_axis(const MropeArgs& a, int i) {
  if (a.interleaved) {  // dealt in turn: axis i % n_axes while that axis has pairs left, axis 0 after
    const int x = i % a.n_axes;
    const int s = x == 1 ? a.sec[1] : (x == 2 ? a.sec[2] : a.sec[3]);
    return x > 0 && i < a.n_axes * s ? x : 0;
  }
  const int b1 = a.sec[0], b2 = b1 + a.sec[1], b3 = b2 + a.sec[2];
  return (i >= b1) + (i >= b2) + (i >= b3);
}

// Eight elements of a row: v[0..3] at dim o1, v[4..7] at dim o2.
struct Chunk {
  float v[8];
};

template <bool VEC>
__device__ __forceinline__ Chunk load_chunk(const float* row, int o1, int o2) {
  Chunk c;
  if constexpr (VEC) {
    const float4 x = *reinterpret_cast<const float4*>(row + o1);
    const float4 y = *reinterpret_cast<const float4*>(row + o2);
    c = Chunk{{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c.v[e] = row[o1 + e];
      c.v[4 + e] = row[o2 + e];
    }
  }
  return c;
}

// VEC: half a multiple of 4 and 16-byte aligned rows, lanes hold pairs as
// above.  Otherwise lane l holds dims 8l .. 8l + 7 and loads partners one by one.
template <int DT, int D, bool VEC>
__global__ __launch_bounds__(kBlock) void mrope_append_kernel(MropeArgs a) {
  constexpr int LPR = D / 8;          // lanes per row
  constexpr int RPB = kBlock / LPR;   // rows per pass of the block
  __shared__ float2 table[kMaxHalf];  // (sin, cos) of the token's pairs
  const int t = blockIdx.x;
  const int l = threadIdx.x % LPR;
  const int rows = a.n_heads + 2 * a.n_kv;
  const int r_end = min(rows, ((int)blockIdx.y + 1) * a.rows_per_block);
  int r = (int)blockIdx.y * a.rows_per_block + threadIdx.x / LPR;

  const int half = a.half, lp = half / 4;  // VEC: lanes of the turned part
  int o1 = 8 * l, o2 = 8 * l + 4;
  bool turns = 8 * l < 2 * half;
  if constexpr (VEC) {
    turns = l < lp;
    o1 = turns ? 4 * l : 2 * half + 8 * (l - lp);
    o2 = turns ? half + 4 * l : o1 + 4;
  }
  auto source = [&](int row) -> const float* {
    if (row < a.n_heads) return a.q + ((size_t)t * a.n_heads + row) * D;
    row -= a.n_heads;
    return row < a.n_kv ? a.k_new + ((size_t)t * a.n_kv + row) * D : a.v_new + ((size_t)t * a.n_kv + row - a.n_kv) * D;
  };

  // the first rows and the token's slot are on their way while the table is made
  Chunk next{};
  if (r < r_end) next = load_chunk<VEC>(source(r), o1, o2);
  const int seq = a.tok_seq[t], pos = a.tok_pos[t];
  bool stored = seq >= 0 && seq < a.n_rows && pos >= 0 && pos / kPage < a.bt_stride;
  const uint32_t phys = stored ? a.bt[(size_t)seq * a.bt_stride + pos / kPage] : 0u;
  stored = stored && phys < a.num_pages;  // LNSKV_NO_PAGE or outside the pool: not written
  const size_t slot = (size_t)phys * kPage + (size_t)(pos % kPage);

  if ((int)threadIdx.x < half) {
    const int i = threadIdx.x;
    const int p = a.axis_pos[(size_t)pair_axis(a, i) * a.n_tok + t];
    float sn, cs;
    rope_sincos_f64((double)p * (double)a.inv[i], &sn, &cs);
    table[i] = make_float2(sn, cs);
  }
  __syncthreads();

  for (; r < r_end; r += RPB) {  // lanes of one row agree
    Chunk x = next;
    if (r + RPB < r_end) next = load_chunk<VEC>(source(r + RPB), o1, o2);
    const bool is_q = r < a.n_heads, is_v = r >= a.n_heads + a.n_kv;
    if (!is_v && turns) {
      if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 sc = table[4 * l + e];
          float y0, y1;
          rope_turn(x.v[e], x.v[4 + e], sc.x, sc.y, &y0, &y1);
          x.v[e] = y0;
          x.v[4 + e] = y1;
        }
      } else {
        const float* row = source(r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 8 * l + e;
          if (i < 2 * half) {
            const bool first = i < half;
            const int pi = first ? i : i - half;
            const float p = row[first ? i + half : pi];
            const float2 sc = table[pi];
            float y0, y1;
            rope_turn(first ? x.v[e] : p, first ? p : x.v[e], sc.x, sc.y, &y0, &y1);
            x.v[e] = first ? y0 : y1;
          }
        }
      }
    }
    // q_out may be q: every partner of the row (held by this wave) has been
    // loaded before any lane of it stores
    if constexpr (!VEC) __builtin_amdgcn_wave_barrier();
    if (is_q) {
      float* dst = a.q_out + ((size_t)t * a.n_heads + r) * D;
      if constexpr (VEC) {
        *reinterpret_cast<float4*>(dst + o1) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        *reinterpret_cast<float4*>(dst + o2) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[8 * l + e] = x.v[e];
      }
      continue;
    }
    const int h = r - a.n_heads - (is_v ? a.n_kv : 0);
    uint8_t* pool = is_v ? a.v_pages : a.k_pages;
    const size_t at = (slot * a.n_kv + h) * D;
    if constexpr (DT == LNSKV_DTYPE_F32) {
      float* dst = reinterpret_cast<float*>(pool) + at;
      if (stored) {
        *reinterpret_cast<float4*>(dst + o1) = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        *reinterpret_cast<float4*>(dst + o2) = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
      }
    } else if constexpr (DT == LNSKV_DTYPE_F16) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(pool) + at;
      auto pack = [](float lo, float hi) { return to_f16_bits(lo) | (to_f16_bits(hi) << 16); };
      if (stored) {
        *reinterpret_cast<uint2*>(dst + o1) = make_uint2(pack(x.v[0], x.v[1]), pack(x.v[2], x.v[3]));
        *reinterpret_cast<uint2*>(dst + o2) = make_uint2(pack(x.v[4], x.v[5]), pack(x.v[6], x.v[7]));
      }
    } else {
      float amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x.v[e]));
      amax = group_max<LPR>(amax);
      const float sc = amax == 0.0f ? 1.0f : amax / 127.0f;
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4] |= ((uint32_t)to_q8(x.v[e], sc) & 0xFFu) << (8 * (e & 3));
      if (stored) {
        *reinterpret_cast<uint32_t*>(pool + at + o1) = w[0];
        *reinterpret_cast<uint32_t*>(pool + at + o2) = w[1];
        if (l == 0) (is_v ? a.v_scales : a.k_scales)[slot * a.n_kv + h] = sc;
      }
    }
  }
}

template <int DT, int D>
void launch_mrope_d(const MropeArgs& a, bool vec, dim3 grid, hipStream_t st) {
  if (vec)
    mrope_append_kernel<DT, D, true><<<grid, kBlock, 0, st>>>(a);
  else
    mrope_append_kernel<DT, D, false><<<grid, kBlock, 0, st>>>(a);
}

template <int DT>
void launch_mrope_dt(const MropeArgs& a, int d, bool vec, dim3 grid, hipStream_t st) {
  switch (d) {
    case 64: launch_mrope_d<DT, 64>(a, vec, grid, st); break;
    case 128: launch_mrope_d<DT, 128>(a, vec, grid, st); break;
    default: launch_mrope_d<DT, 256>(a, vec, grid, st); break;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace lnskv

using namespace lnskv;

extern "C" int lnskv_mrope_append(const lnskv_pages* c, const lnskv_rope* rope, const int32_t* sections,
                                  int32_t n_axes, int32_t interleaved, const float* q, float* q_out, int32_t n_heads,
                                  const float* k_new, const float* v_new, const int32_t* axis_pos,
                                  const int32_t* tok_seq, const int32_t* tok_pos, int32_t n_tok, const uint32_t* bt,
                                  int32_t bt_stride, int32_t n_rows, lnskv_stream_t stream) {
  clear_error();
  if (int rc = check_pages(c)) return rc;
  const int d = (int)c->head_dim;
  if (!rope || !rope->inv_freqs_dev)
    return fail(LNSKV_ERR_INVALID, "rope and its inverse frequencies must be non-null");
  if (rope->rotary_dim < 2 || rope->rotary_dim % 2 != 0 || rope->rotary_dim > d)
    return fail(LNSKV_ERR_INVALID, "rotary_dim %d must be even and in [2, head_dim %d]", rope->rotary_dim, d);
  if (!sections || n_axes < 1 || n_axes > kMaxAxes)
    return fail(LNSKV_ERR_INVALID, "sections must be non-null and n_axes %d in [1, %d]", n_axes, kMaxAxes);
  if (interleaved != 0 && interleaved != 1) return fail(LNSKV_ERR_INVALID, "interleaved %d must be 0 or 1", interleaved);
  const int half = rope->rotary_dim / 2;
  MropeArgs a{};
  int64_t sum = 0;
  for (int x = 0; x < n_axes; ++x) {
    if (sections[x] < 0) return fail(LNSKV_ERR_INVALID, "sections[%d] = %d is negative", x, sections[x]);
    a.sec[x] = sections[x];
    sum += sections[x];
    // the last pair dealt to axis x is x + n_axes (sections[x] - 1)
    if (interleaved && x > 0 && sections[x] > 0 && x + (int64_t)n_axes * (sections[x] - 1) >= half)
      return fail(LNSKV_ERR_INVALID, "axis %d cannot be dealt %d of %d pairs in turn with %d axes", x, sections[x], half,
                  n_axes);
  }
  if (sum != half) return fail(LNSKV_ERR_INVALID, "sections sum to %lld, rotary_dim / 2 is %d", (long long)sum, half);
  if (n_tok < 0) return fail(LNSKV_ERR_INVALID, "n_tok %d is negative", n_tok);
  if ((q == nullptr) != (q_out == nullptr)) return fail(LNSKV_ERR_INVALID, "q and q_out go together");
  if (q && (n_heads <= 0 || n_heads > 65536 || n_heads % (int)c->n_kv_heads != 0))
    return fail(LNSKV_ERR_INVALID, "n_heads %d is not a multiple of n_kv_heads %u in [1, 65536]", n_heads, c->n_kv_heads);
  if (n_tok == 0) return LNSKV_OK;
  if (!k_new || !v_new || !axis_pos || !tok_seq || !tok_pos || !bt)
    return fail(LNSKV_ERR_INVALID, "append arguments must be non-null");
  if (bt_stride <= 0) return fail(LNSKV_ERR_INVALID, "bt_stride %d must be positive", bt_stride);
  if (n_rows < 0) return fail(LNSKV_ERR_INVALID, "n_rows %d is negative", n_rows);
  if (q && q != q_out) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(q), y = reinterpret_cast<uintptr_t>(q_out);
    if ((x < y ? y - x : x - y) < (size_t)n_tok * n_heads * d * sizeof(float))
      return fail(LNSKV_ERR_INVALID, "q_out must be q itself or not overlap it");
  }
  a.k_pages = static_cast<uint8_t*>(c->k_pages);
  a.v_pages = static_cast<uint8_t*>(c->v_pages);
  a.k_scales = c->k_scales;
  a.v_scales = c->v_scales;
  a.q = q;
  a.q_out = q_out;
  a.k_new = k_new;
  a.v_new = v_new;
  a.axis_pos = axis_pos;
  a.tok_seq = tok_seq;
  a.tok_pos = tok_pos;
  a.bt = bt;
  a.inv = rope->inv_freqs_dev;
  a.n_axes = n_axes;
  a.interleaved = interleaved;
  a.half = half;
  a.n_tok = n_tok;
  a.n_heads = q ? n_heads : 0;
  a.n_kv = (int32_t)c->n_kv_heads;
  a.n_rows = n_rows;
  a.bt_stride = bt_stride;
  a.num_pages = c->num_pages;
  const int rpb = kBlock / (d / 8), rows = a.n_heads + 2 * a.n_kv;
  const int passes = (rows + rpb - 1) / rpb;
  // a block per token once tokens fill the card (one table a token), else shares of its
  // rows: us, block per token | shares, 128-wide f16: 32 tokens 3.8 | 3.0, 512 6.9 | 6.6,
  // 1024 9.6 | 10.8, 4096 36.7 | 37.5; 256-wide Q8A 4.3 | 3.4, 7.5 | 7.1, 10.2 | 12.6,
  // 36.4 | 41.7
  a.rows_per_block = n_tok >= 1024 ? passes * rpb : rpb;
  const dim3 grid((unsigned)n_tok, (unsigned)((rows + a.rows_per_block - 1) / a.rows_per_block));
  const bool vec = half % 4 == 0 && aligned16(q) && aligned16(q_out) && aligned16(k_new) && aligned16(v_new);
  switch (c->dtype) {
    case LNSKV_DTYPE_F32: launch_mrope_dt<LNSKV_DTYPE_F32>(a, d, vec, grid, (hipStream_t)stream); break;
    case LNSKV_DTYPE_F16: launch_mrope_dt<LNSKV_DTYPE_F16>(a, d, vec, grid, (hipStream_t)stream); break;
    default: launch_mrope_dt<LNSKV_DTYPE_Q8A>(a, d, vec, grid, (hipStream_t)stream); break;
  }
  return hip_check("mrope append kernel launch");
}
