// Decode attention on pages that the f16 matrix products do not take (f32 pages, and
// 64-wide heads of every page type), for the decode variants: both products as
// v_mfma_f32_16x16x4_f32, one wave per page, 16 query rows, no LDS and no exchange
// between lanes but for the maxima.
//
// Lane (g, n) = (lane / 16, lane % 16).  A contraction may take its index in any
// order, as long as both operands take the same, so each operand is what a lane
// loads with wide loads from the page as it lies in memory:
//  S^T[16 tok][16 row] = K . Q^T: the lane holds token n's elements 4 E j + E g + e
//   (E = elements of 16 bytes, load j: 64 bytes of a row per 4 lanes) and the same
//   elements of query row n; product (j, e) contracts over g.  The lane gets the
//   scores of tokens 4g + ii of row n.
//  O[16 row][D] += P . V: product ii contracts over tokens 4g + ii, whose weight
//   for row n the lane already holds.  It loads elements 64 c + 4n + e of that
//   token (a row of V per 16 lanes); product (ii, c, e) gives output columns
//   64 c + 4n + e of rows 4g + i.  A masked token's V is its own lanes' to clear.
// A page takes D / 2 products of 32 cycles whatever its type and head count, against
// which HBM delivers f32 and f16 pages later; Q8A pages of 64-wide heads at about the
// same rate.  24 sequences x 4 kv heads of 8, window 1000 + 21, f32, 64-wide: 13.2 us and
// 4.0 for the merge (44 MB take 9.2 at a large copy's rate); the generic decode kernel's
// vector code took 21.8.  Three sequences of 3700 Q8A tokens 11 us (34: its sums across
// rows at the end of every block).
#pragma once

#include "lnskv_device.h"

namespace lnskv {
namespace {

template <int DT, int D>
struct TileGeo {
  static constexpr int ES = Storage<DT>::kBytes;
  static constexpr int E = 16 / ES;           // elements of a K load
  static constexpr int KL = D / (4 * E);      // K loads of a page
  static constexpr int VW = ES;               // 32-bit words of four elements
  static constexpr int C = D / 64;
};

template <int DT, int D>
struct TilePage {
  using G = TileGeo<DT, D>;
  uint32_t k[G::KL][4];
  uint32_t v[4][G::C][G::VW];
  float ks, vs;  // Q8A: of token 4g + n % 4
};

template <int DT, int D>
struct TileState {
  float q[D / 4];
  float4v acc[D / 16];  // [4 c + e][i]: O[row 4g + i][64 c + 4n + e]
  float m, l;           // of row n (l: over this lane's tokens)
};

template <int DT>
__device__ __forceinline__ float tile_elem(const uint32_t* w, int e) {
  if constexpr (DT == LNSKV_DTYPE_F32) return __builtin_bit_cast(float, w[e]);
  else if constexpr (DT == LNSKV_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> (16 * (e & 1))));
  else return (float)(int8_t)(w[e / 4] >> (8 * (e & 3)));
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// a: the pools (k_pages, v_pages, k_scales, v_scales, n_kv).
template <int DT, int D, class Args>
__device__ __forceinline__ void tile_load(const Args& a, uint32_t phys, int kvh, int g, int n, TilePage<DT, D>& pg) {
  using G = TileGeo<DT, D>;
  const size_t slot = (size_t)phys * kPage;
  const uint8_t* kp = a.k_pages + ((slot + n) * a.n_kv + kvh) * D * G::ES + 16 * g;
#pragma unroll
  for (int j = 0; j < G::KL; ++j) load_words(kp + 64 * j, pg.k[j]);
#pragma unroll
  for (int ii = 0; ii < 4; ++ii) {
    const uint8_t* vp = a.v_pages + (((slot + 4 * g + ii) * a.n_kv + kvh) * D + 4 * n) * G::ES;
#pragma unroll
    for (int c = 0; c < G::C; ++c) load_words(vp + 64 * c * G::ES, pg.v[ii][c]);
  }
  if constexpr (DT == LNSKV_DTYPE_Q8A) {
    const size_t s = (slot + 4 * g + (n & 3)) * a.n_kv + kvh;
    pg.ks = a.k_scales[s];
    pg.vs = a.v_scales[s];
  }
}

// q: row n's D values.
template <int DT, int D>
__device__ __forceinline__ void tile_init(TileState<DT, D>& st, const float* q, float scale, int g) {
  using G = TileGeo<DT, D>;
#pragma unroll
  for (int j = 0; j < G::KL; ++j)
#pragma unroll
    for (int x = 0; x < G::E / 4; ++x) {
      const float4v w = *reinterpret_cast<const float4v*>(q + 4 * G::E * j + G::E * g + 4 * x);
#pragma unroll
      for (int e = 0; e < 4; ++e) st.q[G::E * j + 4 * x + e] = w[e] * scale;
    }
#pragma unroll
  for (int b = 0; b < D / 16; ++b) st.acc[b] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  st.m = kMInit;
  st.l = 0.0f;
}

// One page through the online softmax.  full: every row attends every token.
// Otherwise sees(t) says whether row n attends token t of the page, and any(t)
// whether some row does (where none does, K and V may be any bits).
template <int DT, int D, class Sees, class Any>
__device__ __forceinline__ void tile_consume(TileState<DT, D>& st, TilePage<DT, D>& pg, bool full, int g, Sees sees,
                                             Any any) {
  using G = TileGeo<DT, D>;
  float4v s = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s;
#pragma unroll
  for (int j = 0; j < G::KL; ++j)
#pragma unroll
    for (int e = 0; e < G::E; e += 2) {
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_elem<DT>(pg.k[j], e), st.q[G::E * j + e], s, 0, 0, 0);
      s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_elem<DT>(pg.k[j], e + 1), st.q[G::E * j + e + 1], s2, 0, 0, 0);
    }
  s += s2;
  float vs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  if constexpr (DT == LNSKV_DTYPE_Q8A) {
    s[0] *= dpp_mov<0x00>(pg.ks), s[1] *= dpp_mov<0x55>(pg.ks), s[2] *= dpp_mov<0xAA>(pg.ks), s[3] *= dpp_mov<0xFF>(pg.ks);
    vs[0] = dpp_mov<0x00>(pg.vs), vs[1] = dpp_mov<0x55>(pg.vs), vs[2] = dpp_mov<0xAA>(pg.vs), vs[3] = dpp_mov<0xFF>(pg.vs);
  }
  if (!full) {  // wave-uniform
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      if (!sees(4 * g + ii)) s[ii] = -INFINITY;
      if (!any(4 * g + ii)) {
        if constexpr (DT == LNSKV_DTYPE_Q8A) {
          vs[ii] = 0.0f;
        } else {
#pragma unroll
          for (int c = 0; c < G::C; ++c)
#pragma unroll
            for (int x = 0; x < G::VW; ++x) pg.v[ii][c][x] = 0u;
        }
      }
    }
  }
  const float mx = max_xor16(max_xor32(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
  if (__builtin_amdgcn_ballot_w64(mx > st.m)) {  // wave-uniform
    const float mn = fmaxf(st.m, mx), alpha = fast_exp2(st.m - mn);
    st.m = mn;
    st.l *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ar = __shfl(alpha, 20 * g + i, kWave);  // row 4g + i
#pragma unroll
      for (int b = 0; b < D / 16; ++b) st.acc[b][i] *= ar;
    }
  }
  float p[4];
#pragma unroll
  for (int ii = 0; ii < 4; ++ii) p[ii] = fast_exp2(s[ii] - st.m);
  st.l += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
  for (int ii = 0; ii < 4; ++ii) {
    if constexpr (DT == LNSKV_DTYPE_Q8A) p[ii] *= vs[ii];
#pragma unroll
    for (int c = 0; c < G::C; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        st.acc[4 * c + e] =
            __builtin_amdgcn_mfma_f32_16x16x4f32(p[ii], tile_elem<DT>(pg.v[ii][c], e), st.acc[4 * c + e], 0, 0, 0);
  }
}

// Pages first, first + step, ... below end (at most 64 of them), two in flight.
// phys(i), full(i, valid), and the masks of page i as tile_consume takes them.
template <int DT, int D, class Args, class Phys, class Consume>
__device__ __forceinline__ void tile_pages(const Args& a, int kvh, int g, int n, int first, int step, int end,
                                           Phys phys, Consume consume) {
  TilePage<DT, D> pg[2];
  bool valid[2];
  auto load = [&](int i, int b) {
    const uint32_t ph = phys(i);
    valid[b] = ph < a.num_pages;
    tile_load<DT, D>(a, valid[b] ? ph : 0u, kvh, g, n, pg[b]);  // a missing page reads page 0, masked
  };
  if (first < end) load(first, 0);
  for (int i = first; i < end; i += 2 * step) {
    if (i + step < end) load(i + step, 1);
    consume(i, valid[0], pg[0]);
    if (i + step < end) {
      if (i + 2 * step < end) load(i + 2 * step, 0);
      consume(i + step, valid[1], pg[1]);
    }
  }
}

// Grid (kv head, partition, sequence), four waves: a partition's pages go round to
// the waves, whose rows merge in LDS at the end.  A row is a query head of the
// sequence; columns past the last head repeat them.
template <int DT, int D, int REP, int VAR>
__global__ __launch_bounds__(kBlock) void decode_tile_kernel(DecodeArgs a, VarArgs<VAR> x) {
  __shared__ __attribute__((aligned(16))) EpilogueLds<REP, D> sm;
  const int kvh = blockIdx.x, part = blockIdx.y, s = blockIdx.z;
  const SeqWindow w = seq_window<false, VAR>(a, s, x);
  if (part >= w.nparts) return;  // block-uniform
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, g = lane >> 4, n = lane & 15;
  [[maybe_unused]] SinkSpan sp;
  int ta, tb;  // kSink: counted without the gap
  if constexpr (VAR == kSink) {
    sp = sink_span(x, w.L);
    ta = part * a.split;
    tb = min(max(w.L - sp.gap * kPage, 0), ta + a.split);
  } else {
    ta = w.p0 + part * a.split;
    tb = min(w.L, ta + a.split);
  }
  auto entry = [&](int pg) {
    if constexpr (VAR == kSink) return sink_entry(sp, pg);
    return pg;
  };
  const int pg0 = ta / kPage, pages = ta < tb ? (tb - 1) / kPage + 1 - pg0 : 0;  // at most 64
  int row = s;
  if constexpr (VAR == kPrefix) {
    const PrefixRows pr = prefix_rows(x, s, a.n_heads);
    row = pg0 + lane < pr.pages ? pr.first : s;
  }
  const uint32_t btv = lane < pages ? a.bt[(size_t)row * a.bt_stride + entry(pg0 + lane)] : 0xFFFFFFFFu;
  TileState<DT, D> st;
  tile_init<DT, D>(st, a.q + ((size_t)s * a.n_heads + kvh * REP + n % REP) * D, a.scale_log2, g);
  tile_pages<DT, D>(
      a, kvh, g, n, wave, kWavesPerBlock, pages, [&](int i) { return __builtin_amdgcn_readlane(btv, i); },
      [&](int i, bool valid, TilePage<DT, D>& pg) {
        const int tok0 = entry(pg0 + i) * kPage;
        if constexpr (VAR == kSink) {
          auto sees = [&](int t) { return valid && sink_sees(sp, tok0 + t); };
          tile_consume<DT, D>(st, pg, valid && sink_sees_page(sp, tok0), g, sees, sees);
        } else {
          auto sees = [&](int t) { return valid && tok0 + t < tb; };
          tile_consume<DT, D>(st, pg, valid && tok0 + kPage <= tb, g, sees, sees);
        }
      });
  st.l = sum_xor16(sum_xor32(st.l));
  if (lane < REP) {
    sm.m[wave][lane] = st.m;
    sm.l[wave][lane] = st.l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * g + i < REP) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<float4v*>(&sm.acc[wave][4 * g + i][64 * c + 4 * n]) =
            float4v{st.acc[4 * c][i], st.acc[4 * c + 1][i], st.acc[4 * c + 2][i], st.acc[4 * c + 3][i]};
    }
  __syncthreads();
  finish_block<REP, D, VAR>(a, sm, w, s, kvh, part, x);
}

}  // namespace
}  // namespace lnskv
