// Decode attention on f32 pages and on 64-wide heads of every page type, for the decode
// variants: a wave per page and 16 query rows, no LDS and no exchange between lanes but
// for the maxima.  f32 pages in v_mfma_f32_16x16x4_f32; f16 and Q8A pages (codes are exact
// in f16) in f16 products with q and the weights as hi and lo parts.
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
// f16 products take the same elements eight at a time (scores, over 32 of them) and the
// four tokens of a lane at once (P.V).
// A page takes D / 2 f32 products of 32 cycles, or 4 + 8 f16 products of 16, whatever the
// head count: bound by HBM, or by start-up and the merge where partitions are short.  24
// sequences x 4 kv heads of 8, window 1000 + 21, f32, 64-wide: 13.2 us and 4.0 for the
// merge (44 MB take 9.2 at a large copy's rate); the generic decode kernel's vector code
// took 21.8.  48 x 4 of 3000, f16, 64-wide: 39 us (147 MB, 31).  Sixty sequences of 9400
// tokens behind 9000 shared ones, f16: 44 us with f16 products, 78 with f32 ones.
#pragma once

#include "lnskv_mfma.h"

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

// f16 and Q8A pages (64-wide heads): f16 products, q and the weights as pairs of f16.
template <int DT>
constexpr bool kTileHalf = DT != LNSKV_DTYPE_F32;

template <int DT, int D>
struct TileState {
  float q[kTileHalf<DT> ? 1 : D / 4];
  half8 qh[kTileHalf<DT> ? 2 : 1], ql[kTileHalf<DT> ? 2 : 1];  // q / 2^E, hi and lo
  float qexp;           // 2^E
  float4v acc[D / 16];  // [4 c + e][i]: O[row 4g + i][64 c + 4n + e] (Q8A: over vnorm)
  float m, l;           // of row n (l: over this lane's tokens)
  float vnorm, vinv;    // Q8A: a power of two that follows the largest V scale, and 1 over it
};

template <int DT>
__device__ __forceinline__ float tile_elem(const uint32_t* w, int e) {
  static_assert(!kTileHalf<DT>);
  return __builtin_bit_cast(float, w[e]);
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
  static_assert(!kTileHalf<DT> || D == 64, "two f16 products per page");
  float x[D / 4];
#pragma unroll
  for (int j = 0; j < G::KL; ++j)
#pragma unroll
    for (int y = 0; y < G::E / 4; ++y) {
      const float4v w = *reinterpret_cast<const float4v*>(q + 4 * G::E * j + G::E * g + 4 * y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[G::E * j + 4 * y + e] = w[e] * scale;
    }
  if constexpr (kTileHalf<DT>) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = max_xor16(max_xor32(amax));
    int E = 0;
    if (amax > 0.0f && amax < INFINITY) (void)frexpf(amax, &E);
    const float inv = ldexpf(1.0f, -E);
    st.qexp = ldexpf(1.0f, E);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float y = x[i] * inv;
      const _Float16 hi = (_Float16)y;
      st.qh[i / 8][i % 8] = hi;
      st.ql[i / 8][i % 8] = (_Float16)(y - (float)hi);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 4; ++i) st.q[i] = x[i];
  }
#pragma unroll
  for (int b = 0; b < D / 16; ++b) st.acc[b] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  st.m = kMInit;
  st.l = st.vnorm = st.vinv = 0.0f;
}

// Elements 4 n .. of rows 4g + i, columns 64 c + 4n ..
template <int DT, int D>
__device__ __forceinline__ float4v tile_out(const TileState<DT, D>& st, int c, int i) {
  const float4v o = {st.acc[4 * c][i], st.acc[4 * c + 1][i], st.acc[4 * c + 2][i], st.acc[4 * c + 3][i]};
  return DT == LNSKV_DTYPE_Q8A ? o * st.vnorm : o;
}

// The products of a page of f16 or Q8A: scores of tokens 4g + ii of row n (Q8A: without
// the scales), and P.V.
template <int DT, int D>
__device__ __forceinline__ float4v tile_scores_half(const TileState<DT, D>& st, const TilePage<DT, D>& pg) {
  float4v s = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    half8 k;
    if constexpr (DT == LNSKV_DTYPE_F16) k = __builtin_bit_cast(half8, u32x4{pg.k[j][0], pg.k[j][1], pg.k[j][2], pg.k[j][3]});
    else k = i8x8_to_f16(uint2v{pg.k[0][2 * j], pg.k[0][2 * j + 1]});
    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, st.qh[j], s, 0, 0, 0);
    s2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, st.ql[j], s2, 0, 0, 0);
  }
  return (s + s2) * st.qexp;
}
template <int DT, int D>
__device__ __forceinline__ void tile_pv_half(TileState<DT, D>& st, const TilePage<DT, D>& pg, const float (&p)[4]) {
  half4 ph, pl, v[4];  // v[ii][e]: token 4g + ii, element 4n + e
#pragma unroll
  for (int ii = 0; ii < 4; ++ii) {
    ph[ii] = (_Float16)p[ii];
    pl[ii] = (_Float16)(p[ii] - (float)ph[ii]);
  }
#pragma unroll
  for (int ii = 0; ii < 4; ii += 2) {
    if constexpr (DT == LNSKV_DTYPE_F16) {
      v[ii] = __builtin_bit_cast(half4, uint2v{pg.v[ii][0][0], pg.v[ii][0][1]});
      v[ii + 1] = __builtin_bit_cast(half4, uint2v{pg.v[ii + 1][0][0], pg.v[ii + 1][0][1]});
    } else {
      const half8 x = i8x8_to_f16(uint2v{pg.v[ii][0][0], pg.v[ii + 1][0][0]});
      v[ii] = half4{x[0], x[1], x[2], x[3]};
      v[ii + 1] = half4{x[4], x[5], x[6], x[7]};
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const half4 b = {v[0][e], v[1][e], v[2][e], v[3][e]};
    st.acc[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(ph, b, st.acc[e], 0, 0, 0);
    st.acc[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(pl, b, st.acc[e], 0, 0, 0);
  }
}

// One page through the online softmax.  full: every row attends every token.
// Otherwise sees(t) says whether row n attends token t of the page, and any(t)
// whether some row does (where none does, K and V may be any bits).
template <int DT, int D, class Sees, class Any>
__device__ __forceinline__ void tile_consume(TileState<DT, D>& st, TilePage<DT, D>& pg, bool full, int g, Sees sees,
                                             Any any) {
  using G = TileGeo<DT, D>;
  float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (kTileHalf<DT>) {
    s = tile_scores_half<DT, D>(st, pg);
  } else {
    float4v s2 = s;
#pragma unroll
    for (int j = 0; j < G::KL; ++j)
#pragma unroll
      for (int e = 0; e < G::E; e += 2) {
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_elem<DT>(pg.k[j], e), st.q[G::E * j + e], s, 0, 0, 0);
        s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(tile_elem<DT>(pg.k[j], e + 1), st.q[G::E * j + e + 1], s2, 0, 0, 0);
      }
    s += s2;
  }
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
  if constexpr (DT == LNSKV_DTYPE_Q8A) {  // f16 weights: over a power of two near the largest scale
    const float vmax = max_xor16(max_xor32(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]))));
    if ((vmax > st.vnorm || vmax * 16.0f < st.vnorm) && vmax > 0.0f) {  // wave-uniform
      int e = 0;
      (void)frexpf(vmax, &e);
      if (st.vnorm > 0.0f) {
        const float r = st.vnorm * ldexpf(1.0f, -e);
#pragma unroll
        for (int b = 0; b < D / 16; ++b) st.acc[b] *= r;
      }
      st.vnorm = ldexpf(1.0f, e);
      st.vinv = ldexpf(1.0f, -e);
    }
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      p[ii] *= vs[ii] * st.vinv;
      // one rounded product for both parts: contracted into the conversions, a product
      // beside a tie of f16 rounds to one hi part and is subtracted from another
      asm("" : "+v"(p[ii]));
    }
  }
  if constexpr (kTileHalf<DT>) {
    tile_pv_half<DT, D>(st, pg, p);
  } else {
#pragma unroll
    for (int ii = 0; ii < 4; ++ii)
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
            tile_out<DT, D>(st, c, i);
    }
  __syncthreads();
  finish_block<REP, D, VAR>(a, sm, w, s, kvh, part, x);
}

}  // namespace
}  // namespace lnskv
