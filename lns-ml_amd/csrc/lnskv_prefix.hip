// Decode attention of sequences that share a prefix: the shared pages are read
// once for all query rows of a group, not once per sequence.
//
// softmax over [0, L) splits into the shared part [0, P) and the sequence's
// own [P, L), each a numerator A = sum 2^(s - m) v, a sum l = sum 2^(s - m) and
// a max m (s in log2 units); the two join as
//   out = (2^(m1 - M) A1 + 2^(m2 - M) A2) / (2^(m1 - M) l1 + 2^(m2 - M) l2).
// 1. prefix kernels: work item = (group, tile of the group's query rows, split of its
//    pages, kv head).  A row is one query head of one sequence; all rows of a
//    tile multiply the same K and V.  Each item leaves a partial row (A, m, l)
//    per query row.
// 2. own kernel (f16 and Q8A pages, 128- and 256-wide heads; the generic decode
//    kernel elsewhere): work item = (sequence, kv head, share of its own pages);
//    a sequence with one share merges the prefix's rows and writes its output.
// 3. join kernel, where sequences may have several shares: their rows and the
//    prefix's into the output.
#include "lnskv_decode_mfma.h"
#include "lnskv_decode_var.h"
#include "lnskv_prefill.h"

namespace lnskv {
namespace {

constexpr int kRowsTile = 64;   // query rows per tile of the f32 kernel: four waves of 16
constexpr int kSplitPages = 8;     // fewest pages of a split, matrix-core kernel
constexpr int kSplitPagesF32 = 2;  // f32 kernel
constexpr int kSharePages = 64;    // most pages of a share of a sequence's own
constexpr int kShareMin = 8;

struct PrefixArgs {
  PrefillArgs pf;  // the pools, for the prefill kernel's page pipeline
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scales;
  const float* v_scales;
  const float* q;         // [n_seq][n_heads][D]
  const uint32_t* bt;     // [n_seq][bt_stride]
  const int32_t* kv_len;  // [n_seq]
  float* part_acc;        // partial rows [group][its sequence][head][split]
  float* part_ml;
  int32_t bt_stride;
  int32_t n_kv;
  int32_t n_heads;
  int32_t rep;
  int32_t max_kv_len;
  int32_t split_pages;  // pages per split
  int32_t n_groups;
  uint32_t num_pages;
  float scale_log2;
  PrefixGroup g[LNSKV_PREFIX_MAX_GROUPS];
};

__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Item `i` of the launch (without its kv head): group, row tile and split, and
// the partial rows of the groups before it.
struct PrefixItem {
  int group, tile, split, splits;
  size_t part0;  // first partial row of the group
};
__device__ __forceinline__ PrefixItem prefix_item(const PrefixArgs& a, int i, int tile_rows) {
  PrefixItem it{-1, 0, 0, 1, 0};
  for (int g = 0; g < a.n_groups; ++g) {  // block-uniform
    const int rows = (a.g[g].end - a.g[g].first) * a.rep;
    const int tiles = ceil_div(rows, tile_rows), splits = ceil_div(a.g[g].pages, a.split_pages);
    if (i < tiles * splits) {  // the tiles of one split side by side: they read the same pages
      it.group = g;
      it.split = i / tiles;
      it.tile = i - it.split * tiles;
      it.splits = splits;
      return it;
    }
    i -= tiles * splits;
    it.part0 += (size_t)rows * a.n_kv * splits;
  }
  return it;
}

// Where row (sequence s, query head h) of an item goes.
struct RowOut {
  float* acc;
  float* ml;
};
template <int D>
__device__ __forceinline__ RowOut row_out(const PrefixArgs& a, const PrefixItem& it, int s, int h) {
  const size_t r = it.part0 + ((size_t)(s - a.g[it.group].first) * a.n_heads + h) * it.splits + it.split;
  return {a.part_acc + r * D, a.part_ml + 2 * r};
}

// Tokens of the prefix that sequence s attends: all of them unless its length
// ends inside; none for a length out of range.
__device__ __forceinline__ int row_tokens(const PrefixArgs& a, int s, int pages) {
  const int L = a.kv_len[s];
  return L > min(a.max_kv_len, a.bt_stride * kPage) ? 0 : min(max(L, 0), pages * kPage);
}

// ---------------------------------------------------------------------------
// f32 pages, and 64-wide heads on every page type, in f32: both products as v_mfma_f32_16x16x4_f32
// over a page of K and V held in LDS as f32 (Q8A: code x scale).  Wave w holds
// rows 16w .. 16w + 15 of the tile.  Lane (g, n) = (lane / 16, lane % 16):
//  S^T[16 tok][16 row] = K . Q^T, product (jj, e) over dims 16 jj + 4 g' + e
//  (g' = 0..3 the contraction index), so that both operands of four products
//  are one 16-byte read; lane (g, n) gets tokens 4g + ii of row n.
//  O[16 row][D] += P . V, product ii over tokens 4 g' + ii: its A operand is the
//  lane's own weight ii; lane (g, n) accumulates O[row 4g + i][16 nb + n].
// LDS rows are D + 4 floats: four rows apart fall 16 banks apart.
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void prefix_f32_kernel(PrefixArgs a) {
  constexpr int ES = Storage<DT>::kBytes;
  constexpr int kStride = D + 4;
  constexpr int kElems = D / 16;              // elements of a row per thread
  constexpr int kWords = kElems * ES / 4;     // and their 32-bit words (1 to 16)
  __shared__ __attribute__((aligned(16))) float ks_[kPage * kStride];
  __shared__ __attribute__((aligned(16))) float vs_[kPage * kStride];
  __shared__ int most_[kWavesPerBlock];
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv);
  const PrefixItem it = prefix_item(a, (int)(blockIdx.x / (unsigned)a.n_kv), kRowsTile);
  if (it.group < 0) return;  // block-uniform
  const PrefixGroup gr = a.g[it.group];
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane >> 4, n = lane & 15;
  const int rows = (gr.end - gr.first) * a.rep;
  const int r0 = it.tile * kRowsTile + 16 * w;  // this wave's first row
  const int pg0 = it.split * a.split_pages, pg_end = min(gr.pages, pg0 + a.split_pages);

  const int rn = min(r0 + n, rows - 1);  // past the last row: that row again, never written
  const int sn = gr.first + rn / a.rep, hn = kvh * a.rep + rn % a.rep;
  const int limit = row_tokens(a, sn, gr.pages);
  // tokens past every row's length are masked in the whole tile: their V is
  // zeroed, since 0 * NaN of a stale slot would reach the sums
  int most = limit;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor(most, o, kWave));
  if (lane == 0) most_[w] = most;
  __syncthreads();
  most = max(max(most_[0], most_[1]), max(most_[2], most_[3]));
  const int pg1 = min(pg_end, (most + kPage - 1) / kPage);
  float4v q[D / 16];
  {
    const float4v* src = reinterpret_cast<const float4v*>(a.q + ((size_t)sn * a.n_heads + hn) * D) + g;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = src[4 * j] * a.scale_log2;
  }
  float4v acc[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) acc[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kMInit, l = 0.0f;

  // this thread's elements of a page: kElems of token threadIdx.x / 16
  const int tt = threadIdx.x >> 4, tc = (threadIdx.x & 15) * kElems;
  uint32_t kw[kWords], vw[kWords];
  float ksc = 1.0f, vsc = 1.0f;
  bool ok = false;
  const uint32_t* bt_row = a.bt + (size_t)gr.first * a.bt_stride;
  auto load = [&](int pg) {
    const uint32_t ph = pg < a.bt_stride ? bt_row[pg] : 0xFFFFFFFFu;
    ok = ph < a.num_pages;
    const size_t slot = (size_t)(ok ? ph : 0u) * kPage + tt;  // a missing page reads page 0, masked
    const size_t off = ((slot * a.n_kv + kvh) * D + tc) * ES;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(a.k_pages + off);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(a.v_pages + off);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      kw[i] = kp[i];
      vw[i] = vp[i];
    }
    if constexpr (DT == LNSKV_DTYPE_Q8A) {
      ksc = a.k_scales[slot * a.n_kv + kvh];
      vsc = a.v_scales[slot * a.n_kv + kvh];
    }
  };
  auto value = [](const uint32_t* word, int e, float sc) -> float {
    const uint32_t x = word[e * ES / 4];
    if constexpr (DT == LNSKV_DTYPE_F32) return __builtin_bit_cast(float, x);
    else if constexpr (DT == LNSKV_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(x >> (16 * (e & 1))));
    else return (float)(int8_t)(x >> (8 * (e & 3))) * sc;
  };
  if (pg0 < pg1) load(pg0);
  for (int pg = pg0; pg < pg1; ++pg) {
    const bool valid = ok;
    __syncthreads();  // every wave is done with the page before
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
      ks_[tt * kStride + tc + e] = value(kw, e, ksc);
      vs_[tt * kStride + tc + e] = valid && pg * kPage + tt < most ? value(vw, e, vsc) : 0.0f;
    }
    __syncthreads();
    if (pg + 1 < pg1) load(pg + 1);
    float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const float4v k = *reinterpret_cast<const float4v*>(ks_ + n * kStride + 16 * j + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[j][e], s, 0, 0, 0);
    }
    const int tok0 = pg * kPage;
#pragma unroll
    for (int ii = 0; ii < 4; ++ii)
      if (!(valid && tok0 + 4 * g + ii < limit)) s[ii] = -INFINITY;
    float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    mx = max_xor16(max_xor32(mx));  // over the page's tokens, row n
    if (__builtin_amdgcn_ballot_w64(mx > m)) {  // wave-uniform
      const float mn = fmaxf(m, mx), alpha = fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ar = __shfl(alpha, 20 * g + i, kWave);  // row 4g + i
#pragma unroll
        for (int nb = 0; nb < D / 16; ++nb) acc[nb][i] *= ar;
      }
    }
    float p[4];
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) p[ii] = fast_exp2(s[ii] - m);
    l += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
    for (int ii = 0; ii < 4; ++ii)
#pragma unroll
      for (int nb = 0; nb < D / 16; ++nb)
        acc[nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[ii], vs_[(4 * g + ii) * kStride + 16 * nb + n], acc[nb], 0, 0, 0);
  }
  l = sum_xor16(sum_xor32(l));
  if (lane < 16 && r0 + n < rows) {
    const RowOut o = row_out<D>(a, it, sn, hn);
    o.ml[0] = m;
    o.ml[1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * g + i;
    if (r < rows) {
      const RowOut o = row_out<D>(a, it, gr.first + r / a.rep, kvh * a.rep + r % a.rep);
#pragma unroll
      for (int nb = 0; nb < D / 16; ++nb) o.acc[16 * nb + n] = acc[nb][i];
    }
  }
}

// ---------------------------------------------------------------------------
// f16 and Q8A pages with 128- or 256-wide heads, on the matrix cores: the
// prefill kernel's page pipeline (eight waves, pairs of pages by DMA through an
// LDS ring, q and the weights as pairs of f16) with query rows gathered from the
// group's sequences.  Every row attends every token of the split, but for rows
// whose length ends inside it.  Column n of wave w holds HW query heads of one
// sequence (column u of the group: sequence u / (rep / HW), heads HW (u % (rep /
// HW)) ..), so that its HW rows have the same length.  HW = 2 shares each K and V
// operand read from LDS between two rows' tiles (NH = 1; a 256-wide head's
// accumulators leave room for one).
template <bool Q8, int NH, int HW>
__global__ __launch_bounds__(kWave * 8) void prefix_mfma_kernel(PrefixArgs a) {
  constexpr int D = NH * kD, NW = 8;
  constexpr int kBatch = NH == 2 ? 1 : 2, kDepth = 3 * kBatch;
  constexpr int RPW = Q8 ? NH + 2 : 16 * NH / NW;  // vector-memory instructions per wave and pair
  constexpr int kRingSlot = Q8 ? kPfQ8Slot<NH> : kPfSlot<NH>;
  __shared__ __attribute__((aligned(16))) uint8_t ring_[kDepth * kRingSlot];
  __shared__ __attribute__((aligned(16))) uint8_t f16buf_[Q8 ? 2 * kBatch * kPfSlot<NH> : 16];
  __shared__ int most_[NW];
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv);
  const PrefixItem it = prefix_item(a, (int)(blockIdx.x / (unsigned)a.n_kv), 16 * NW * HW);
  if (it.group < 0) return;  // block-uniform
  const PrefixGroup gr = a.g[it.group];
  const int lane = (int)(threadIdx.x & (kWave - 1)), w = (int)(threadIdx.x / kWave);
  const int g = lane >> 4, n = lane & 15;
  const int per = a.rep / HW;                        // columns of a sequence
  const int cols = (gr.end - gr.first) * per;
  const int u0 = (it.tile * NW + w) * 16;            // this wave's first column
  const bool active = u0 < cols;
  // past the last column: that column again, never written
  const int un = min(u0 + n, cols - 1);
  const int sn = gr.first + un / per, hn = kvh * a.rep + un % per * HW;
  const int limit = row_tokens(a, sn, gr.pages);  // tokens that column n attends
  int most = limit, least = limit;

  float4v qraw[HW][8 * NH];
#pragma unroll
  for (int hh = 0; hh < HW; ++hh) {
    const float4v* src = reinterpret_cast<const float4v*>(a.q + ((size_t)sn * a.n_heads + hn + hh) * D + 8 * g);
#pragma unroll
    for (int j = 0; j < 4 * NH; ++j) {
      qraw[hh][2 * j] = src[8 * j];
      qraw[hh][2 * j + 1] = src[8 * j + 1];
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    most = max(most, __shfl_xor(most, o, kWave));
    least = min(least, __shfl_xor(least, o, kWave));
  }
  if (lane == 0) most_[w] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) most = max(most, most_[i]);
  const int pg_first = it.split * a.split_pages;
  const int ta = pg_first * kPage, tb = min(min(gr.pages, pg_first + a.split_pages) * kPage, most);
  const int npg = ta < tb ? (tb - 1) / kPage - pg_first + 1 : 0;
  const int npairs = (npg + 1) / 2;

  const uint32_t* bt_row = a.bt + (size_t)gr.first * a.bt_stride;
  int base = pg_first;
  uint32_t btv = 0;
  auto load_window = [&]() {
    const int e = base + lane;
    btv = e < a.bt_stride ? bt_row[e] : 0xFFFFFFFFu;
    wait_vmcnt<0>();
  };
  load_window();
  auto phys_of = [&](int i) -> uint32_t {  // i increases from call to call
    int idx = pg_first + i - base;
    if (idx >= 64) {
      base += 64;
      idx -= 64;
      load_window();
    }
    return __builtin_amdgcn_readlane(btv, idx);
  };

  PfLanes pl;
  const uint32_t rs = (uint32_t)a.n_kv * (NH * kRowBytes);
  const uint32_t page_bytes = kPage * rs;
  const uint32_t kvh_off = (uint32_t)kvh * (NH * kRowBytes);
  {
    const int j = w & 3;  // this wave's quarter of a page region
    const uint32_t R = 4u * (uint32_t)j + (uint32_t)g;
    pl.koff = R * rs + 16u * ((uint32_t)n ^ R);
    pl.voff = (uint32_t)(4 * g + j) * rs + 16u * ((uint32_t)n ^ v_swz((int)R));
    pl.lds_q = 1024u * (uint32_t)j;
    pl.krow = (uint32_t)n * kRowBytes + 16u * ((uint32_t)g ^ ((uint32_t)n & 3u));
    pl.kx = 64u * ((uint32_t)n >> 2);
    const int Rv = 4 * (n >> 2) + g;
    pl.vrow = (uint32_t)Rv * kRowBytes + 8u * (n & 1) + 16u * (uint32_t)((n & 3) >> 1);
    pl.vx = 16u * v_swz(Rv);
  }
  lds_u8* ring = (lds_u8*)ring_;
  uint32_t vbits = 0;  // validity of the ring slots' pages
  auto issue = [&](int i) {
    const int sl = i % kDepth;
    const uint32_t ph0 = phys_of(2 * i);
    const uint32_t ph1 = 2 * i + 1 < npg ? phys_of(2 * i + 1) : 0xFFFFFFFFu;
    const uint32_t bits = (ph0 < a.num_pages ? 1u : 0u) | (ph1 < a.num_pages ? 2u : 0u);
    vbits = (vbits & ~(3u << (2 * sl))) | (bits << (2 * sl));
    if constexpr (Q8)
      pf_issue_q8<NH, true>(a.pf, (uint32_t)a.n_kv * D, (uint32_t)kvh, ring + sl * kRingSlot, ph0, ph1, w);
    else
      pf_issue<RPW>(a.pf, pl, page_bytes, kvh_off, ring + sl * kRingSlot, ph0, ph1, w);
  };
#pragma unroll
  for (int i = 0; i < 2 * kBatch; ++i)
    if (i < npairs) issue(i);

  half8 qh[HW][4 * NH], ql[HW][4 * NH];
  float qexp[HW], m[HW], l[HW];
  float4v acc[HW][8 * NH];
  float vnorm = 0.0f;  // Q8: acc is in units of vnorm
#pragma unroll
  for (int hh = 0; hh < HW; ++hh) {
    float amax = 0.0f;
#pragma unroll
    for (int r = 0; r < 8 * NH; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(qraw[hh][r][e] * a.scale_log2));
    amax = max_xor16(max_xor32(amax));
    int E = 0;
    if (amax > 0.0f && amax < INFINITY) (void)frexpf(amax, &E);
    const float inv = ldexpf(1.0f, -E);
    qexp[hh] = ldexpf(1.0f, E);
#pragma unroll
    for (int j = 0; j < 4 * NH; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = qraw[hh][2 * j + (e >> 2)][e & 3] * a.scale_log2 * inv;
        const _Float16 hi = (_Float16)y;
        qh[hh][j][e] = hi;
        ql[hh][j][e] = (_Float16)(y - (float)hi);
      }
    m[hh] = kMInit;
    l[hh] = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 8 * NH; ++nb) acc[hh][nb] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  }

  for (int i0 = 0; i0 < npairs; i0 += kBatch) {
    const int later = min(max(npairs - (i0 + kBatch), 0), kBatch);  // pairs that may stay in flight
    if (later == 2)
      wait_vmcnt<2 * RPW>();
    else if (later == 1)
      wait_vmcnt<RPW>();
    else
      wait_vmcnt<0>();
    lds_u8* f16b = (lds_u8*)f16buf_ + ((i0 / kBatch) & 1) * (kBatch * kPfSlot<NH>);
    if constexpr (Q8) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (i0 + k < npairs) pf_convert_q8<NH>(ring + ((i0 + k) % kDepth) * kRingSlot, f16b + k * kPfSlot<NH>, w);
    }
    pf_barrier();  // every wave's quarters of this batch landed; the previous batch is consumed
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i0 + 2 * kBatch + k < npairs) issue(i0 + 2 * kBatch + k);
    for (int i = i0; i < min(i0 + kBatch, npairs); ++i) {
      if (active) {
        const int sl = i % kDepth;
        lds_u8* sp = Q8 ? f16b + (i - i0) * kPfSlot<NH> : ring + sl * kRingSlot;
        const lds_u8* sc = ring + sl * kRingSlot + kPfCodeSlot<NH> + w * kPfScaleWave;
        const bool v0 = (vbits >> (2 * sl)) & 1u, v1 = (vbits >> (2 * sl + 1)) & 1u;
        const int tok0 = (pg_first + 2 * i) * kPage;
        const bool whole = v0 && v1 && tok0 + 2 * kPage <= tb;
        // 256-wide heads: no mask-free copy (its register allocation spilled)
        if (NH == 1 && whole && tok0 + 2 * kPage <= least)
          pf_consume<HW, 0, Q8, NH>(acc, m, l, qh, ql, qexp, pl, sp, tok0, v0, v1, ta, tb, limit - 1, ta, true, g, n, sc, &vnorm);
        else if (NH == 2 && whole)
          pf_consume<HW, 1, Q8, NH>(acc, m, l, qh, ql, qexp, pl, sp, tok0, v0, v1, ta, tb, limit - 1, ta, true, g, n, sc, &vnorm);
        else
          pf_consume<HW, 2, Q8, NH>(acc, m, l, qh, ql, qexp, pl, sp, tok0, v0, v1, ta, tb, limit - 1, ta, true, g, n, sc, &vnorm);
      }
    }
  }
  if (!active) return;
#pragma unroll
  for (int hh = 0; hh < HW; ++hh) {
    const float lt = sum_xor16(sum_xor32(l[hh]));
    if (lane < 16 && u0 + n < cols) {
      int u = u0 + n;
      asm volatile("" : "+v"(u));  // sequence and head again, not held through the loop
      const RowOut o = row_out<D>(a, it, gr.first + u / per, kvh * a.rep + u % per * HW + hh);
      o.ml[0] = m[hh];
      o.ml[1] = lt;
    }
#pragma unroll
    for (int ii = 0; ii < 4; ++ii) {
      const int u = u0 + 4 * g + ii;
      if (u < cols) {
        const RowOut o = row_out<D>(a, it, gr.first + u / per, kvh * a.rep + u % per * HW + hh);
#pragma unroll
        for (int nb = 0; nb < 8 * NH; ++nb) o.acc[16 * nb + n] = Q8 ? acc[hh][nb][ii] * vnorm : acc[hh][nb][ii];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The sequences' own pages [P, L).  A workgroup takes one share (at most
// share_pages pages) of one (sequence, kv head); its four waves split the share
// and stream their pages as the decode kernels do, each by itself (K to registers,
// V through an LDS ring, two pages in flight), leave partial rows in LDS, and
// merge them head by head.  No workgroup depends on another.
struct OwnArgs {
  VarArgs<kPrefix> prefix;
  float* own_acc;  // [n_seq][n_heads][shares][D], where a sequence has several shares
  float* own_ml;
  int32_t n_seq;
  int32_t shares;  // of a sequence at most
  int32_t share_pages;
};

// Pages of sequence s past its prefix, and how many shares they make.
struct OwnSpan {
  int L, p0, pages, shares;
  PrefixRows prefix;
};
__device__ __forceinline__ OwnSpan own_span(const DecodeArgs& a, const OwnArgs& x, int s) {
  OwnSpan o;
  int L = a.kv_len[s];
  o.L = L > min(a.max_kv_len, a.bt_stride * kPage) ? 0 : max(L, 0);
  o.prefix = prefix_rows(x.prefix, s, a.n_heads);
  o.p0 = min(o.prefix.pages * kPage, o.L);
  o.pages = o.L > o.p0 ? (o.L - 1) / kPage - o.p0 / kPage + 1 : 0;
  o.shares = max(1, ceil_div(o.pages, x.share_pages));
  return o;
}

// Merges rows [r0, r0 + n) of (acc, ml) into (M, Ls, A): lane l holds columns
// l + 64 c; eight rows' loads in flight.
template <int D>
__device__ __forceinline__ void merge_rows(const float* acc, const float* ml, size_t r0, int n, float& M, float& Ls,
                                           float (&A)[D / kWave]) {
  constexpr int C = D / kWave;
  float m2, l2, a2[C];
  merge_wave<D, 1, 8>(reinterpret_cast<const float2*>(ml), acc, 0, n, [=](int j) { return r0 + (size_t)j; }, m2, l2, a2);
  const float Mn = fmaxf(M, m2), wa = fast_exp2(M - Mn), wb = fast_exp2(m2 - Mn);
  M = Mn;
  Ls = Ls * wa + l2 * wb;
#pragma unroll
  for (int c = 0; c < C; ++c) A[c] = A[c] * wa + a2[c] * wb;
}

constexpr int kOwnWaves = 4;

template <int REP, bool Q8, int NH>
__global__ __launch_bounds__(kWave* kOwnWaves) __attribute__((amdgpu_waves_per_eu(NH == 1 ? 2 : 1)))
void prefix_own_kernel(DecodeArgs a, OwnArgs x) {
  constexpr int NW = kOwnWaves, D = NH * kD, C = D / kWave, kRow = D + 2;
  constexpr int kSlots = Q8 ? 1 : 2;
  typedef __attribute__((address_space(3))) float lds_f32;
  __shared__ __attribute__((aligned(16))) uint8_t vring_[NW][kSlots * NH * kVSlot];
  __shared__ __attribute__((aligned(16))) float part_[NW * REP * kRow];
  const int wi = (int)(threadIdx.x / kWave), lane = (int)(threadIdx.x % kWave);
  // share slowest: the first shares, which every sequence has, start first
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv);
  const int s = (int)(blockIdx.x / (unsigned)a.n_kv % (unsigned)x.n_seq);
  const int share = (int)(blockIdx.x / (unsigned)a.n_kv / (unsigned)x.n_seq);
  const OwnSpan o = own_span(a, x, s);
  if (share >= o.shares) return;  // block-uniform
  const int lo = (int)((int64_t)o.pages * share / o.shares), hi = (int)((int64_t)o.pages * (share + 1) / o.shares);
  // wave w: pages [lo + w per, lo + (w + 1) per) of the sequence's own
  const int per = ceil_div(hi - lo, NW);
  const int i0 = min(hi, lo + wi * per), i1 = min(hi, i0 + per);
  if (i0 < i1) {
    const int pg0 = o.p0 / kPage;
    PieceLoads<REP, NH> pl;
    piece_loads<REP, false, false, Q8, NH>(a, s, kvh, pg0 + i0, pl);
    PieceOut po;
    po.final = false;
    po.pbase = (size_t)wi * REP;
    po.pstride = 1;
    po.in_lds = true;
    po.lds = (lds_f32*)part_;
    if constexpr (Q8)
      run_piece_q8<REP, 2, false, NH, false>(a, (lds_u8*)vring_[wi], (lds_u8*)vring_[wi], pl, true, s, kvh,
                                             (pg0 + i0) * kPage, min(o.L, (pg0 + i1) * kPage), false, o.L - 1, po, nullptr);
    else
      run_piece<REP, false, 2, false, NH>(a, (lds_u8*)vring_[wi], (lds_u8*)vring_[wi], pl, true, s, kvh,
                                          (pg0 + i0) * kPage, min(o.L, (pg0 + i1) * kPage), false, o.L - 1, po, nullptr);
  }
  __syncthreads();
  const int nw = hi > lo ? ceil_div(hi - lo, per) : 0;  // waves that left rows
  for (int h = wi; h < REP; h += NW) {  // wave-uniform
    const size_t hrow = (size_t)s * a.n_heads + (size_t)kvh * REP + h;
    float M = kMInit, Ls = 0.0f, A[C];
#pragma unroll
    for (int c = 0; c < C; ++c) A[c] = 0.0f;
    for (int w = 0; w < nw; ++w) {
      const lds_f32* row = (const lds_f32*)part_ + ((size_t)w * REP + h) * kRow;
      const float m = row[D], Mn = fmaxf(M, m);
      const float wa = fast_exp2(M - Mn), wb = fast_exp2(m - Mn);
      Ls = Ls * wa + row[D + 1] * wb;
#pragma unroll
      for (int c = 0; c < C; ++c) A[c] = A[c] * wa + row[lane + c * kWave] * wb;
      M = Mn;
    }
    if (o.shares == 1) {
      merge_rows<D>(x.prefix.part_acc, x.prefix.part_ml, o.prefix.base + (size_t)(kvh * REP + h) * o.prefix.splits,
                    o.prefix.splits, M, Ls, A);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const size_t i = hrow * D + c * kWave + lane;
        a.out[i] = gated(a, i, Ls > 0.0f ? A[c] / Ls : 0.0f);
      }
    } else {
      const size_t r = hrow * x.shares + share;
#pragma unroll
      for (int c = 0; c < C; ++c) x.own_acc[r * D + c * kWave + lane] = A[c];
      if (lane == 0) {
        x.own_ml[2 * r] = M;
        x.own_ml[2 * r + 1] = Ls;
      }
    }
  }
}

// The outputs of the sequences with several shares: wave per (sequence, head).
template <int D>
__global__ __launch_bounds__(kBlock) void prefix_join_kernel(DecodeArgs a, OwnArgs x) {
  constexpr int C = D / kWave;
  const int64_t i = (int64_t)blockIdx.x * kWavesPerBlock + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (i >= (int64_t)x.n_seq * a.n_heads) return;
  const int s = __builtin_amdgcn_readfirstlane((int)(i / a.n_heads));
  const int h = __builtin_amdgcn_readfirstlane((int)(i - (int64_t)s * a.n_heads));
  const OwnSpan o = own_span(a, x, s);
  if (o.shares == 1) return;
  float M = kMInit, Ls = 0.0f, A[C];
#pragma unroll
  for (int c = 0; c < C; ++c) A[c] = 0.0f;
  merge_rows<D>(x.own_acc, x.own_ml, (size_t)i * x.shares, o.shares, M, Ls, A);
  merge_rows<D>(x.prefix.part_acc, x.prefix.part_ml, o.prefix.base + (size_t)h * o.prefix.splits, o.prefix.splits, M,
                Ls, A);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const size_t e = (size_t)i * D + c * kWave + lane;
    a.out[e] = gated(a, e, Ls > 0.0f ? A[c] / Ls : 0.0f);
  }
}

template <bool Q8, int NH>
void launch_own_rep(const DecodeArgs& a, const OwnArgs& x, int rep, unsigned blocks, hipStream_t st) {
  switch (rep) {
    case 1: prefix_own_kernel<1, Q8, NH><<<blocks, kWave * kOwnWaves, 0, st>>>(a, x); break;
    case 2: prefix_own_kernel<2, Q8, NH><<<blocks, kWave * kOwnWaves, 0, st>>>(a, x); break;
    case 4: prefix_own_kernel<4, Q8, NH><<<blocks, kWave * kOwnWaves, 0, st>>>(a, x); break;
    default: prefix_own_kernel<8, Q8, NH><<<blocks, kWave * kOwnWaves, 0, st>>>(a, x); break;
  }
}

template <bool Q8>
void launch_prefix_mfma(const PrefixArgs& a, int d, int tile_rows, unsigned blocks, hipStream_t st) {
  if (d == 256)
    prefix_mfma_kernel<Q8, 2, 1><<<blocks, kWave * 8, 0, st>>>(a);
  else if (tile_rows == 256)
    prefix_mfma_kernel<Q8, 1, 2><<<blocks, kWave * 8, 0, st>>>(a);
  else
    prefix_mfma_kernel<Q8, 1, 1><<<blocks, kWave * 8, 0, st>>>(a);
}

template <int DT>
void launch_prefix_f32(const PrefixArgs& a, int d, unsigned blocks, hipStream_t st) {
  switch (d) {
    case 64: prefix_f32_kernel<DT, 64><<<blocks, kBlock, 0, st>>>(a); return;
    default: break;
  }
  if constexpr (DT == LNSKV_DTYPE_F32) {
    if (d == 128)
      prefix_f32_kernel<DT, 128><<<blocks, kBlock, 0, st>>>(a);
    else
      prefix_f32_kernel<DT, 256><<<blocks, kBlock, 0, st>>>(a);
  }
}

// ---------------------------------------------------------------------------
// The host's view of a call.
struct PrefixPlan {
  VarPlan own;            // the generic kernel over the sequences' own pages
  int shares = 0;         // own kernel: shares of a sequence at most (0: the generic kernel)
  int share_pages = 0;
  int split_pages = 1;
  int tile_rows = 0;      // query rows of a work item
  int64_t items = 0;      // work items per kv head
  int64_t part_rows = 0;  // partial rows of the prefixes
  size_t own_at = 0, part_at = 0, ws_bytes = 0;
  int n_groups = 0;
  PrefixGroup g[LNSKV_PREFIX_MAX_GROUPS];
};

int plan_prefix(const lnskv_pages* c, const int32_t* groups, int n_groups, int n_seq, int n_heads, int max_kv_len,
                PrefixPlan* p) {
  if (n_groups < 0 || n_groups > LNSKV_PREFIX_MAX_GROUPS)
    return fail(LNSKV_ERR_INVALID, "n_groups %d out of range [0, %d]", n_groups, LNSKV_PREFIX_MAX_GROUPS);
  if (n_groups > 0 && !groups) return fail(LNSKV_ERR_INVALID, "groups must be non-null");
  const int rep = n_heads / (int)c->n_kv_heads, d = (int)c->head_dim;
  // the matrix-core kernel takes two heads of a sequence per column where some
  // group has more than 128 rows
  int most_rows = 0;
  for (int i = 0; i < n_groups; ++i) most_rows = std::max(most_rows, std::min(groups[3 * i + 1], n_seq) * rep);
  p->tile_rows = !var_mfma(c) ? kRowsTile : (d == 128 && rep > 1 && most_rows > 128 ? 256 : 128);
  const int64_t all = (int64_t)max_kv_len / kPage + 1;
  int64_t own_pages = 0, most = 0, tiles = 0, max_shared = 0;  // summed over sequences; of one sequence
  int at = 0;
  for (int i = 0; i < n_groups; ++i) {
    const int first = groups[3 * i], n = groups[3 * i + 1], tok = groups[3 * i + 2];
    if (first < at || n <= 0 || n > n_seq - first || tok < 0)
      return fail(LNSKV_ERR_INVALID,
                  "group %d {%d, %d, %d}: groups lie in [0, %d), in order and apart, with tokens >= 0", i, first, n, tok,
                  n_seq);
    if (first > at) most = all;
    own_pages += (first - at) * all;
    at = first + n;
    const int64_t shared = std::min<int64_t>(tok / kPage, all);
    own_pages += n * std::max<int64_t>(all - shared, 1);
    most = std::max(most, std::max<int64_t>(all - shared, 1));
    if (shared == 0) continue;
    p->g[p->n_groups++] = PrefixGroup{first, at, (int32_t)shared};
    tiles += ceil_div(n * rep, p->tile_rows);
    max_shared = std::max(max_shared, shared);
  }
  if (at < n_seq) most = all;
  own_pages += (n_seq - at) * all;
  const size_t row = ((size_t)d + 2) * sizeof(float);
  if (var_mfma(c)) {
    // shares of at most kSharePages pages, fewer where that leaves compute units idle
    const int64_t units = own_pages * c->n_kv_heads;
    p->share_pages = n_seq * (int64_t)c->n_kv_heads >= 256
                         ? kSharePages
                         : (int)std::min<int64_t>(kSharePages, std::max<int64_t>(kShareMin, (units + 511) / 512));
    p->shares = (int)std::max<int64_t>(1, (most + p->share_pages - 1) / p->share_pages);
    if ((int64_t)p->shares * n_seq * c->n_kv_heads > INT32_MAX)
      return fail(LNSKV_ERR_UNSUPPORTED, "a batch of more than 2^31 shares");
    p->own_at = kWsHeaderBytes;
    p->ws_bytes = p->shares > 1 ? kWsHeaderBytes + (size_t)p->shares * n_seq * n_heads * row : 0;
  } else {
    if (int rc = plan_generic(c, n_seq, n_heads, most, &p->own)) return rc;
    p->ws_bytes = p->own.ws_bytes;
  }
  if (p->n_groups == 0) return LNSKV_OK;
  // splits of equal pages, about one matrix-core item or two of the f32 kernel's per
  // compute unit
  const int64_t want = std::max<int64_t>(1, (var_mfma(c) ? 256 : 512) / (tiles * c->n_kv_heads));
  p->split_pages = (int)std::max<int64_t>(var_mfma(c) ? kSplitPages : kSplitPagesF32, (max_shared + want - 1) / want);
  for (int i = 0; i < p->n_groups; ++i) {
    const int64_t n = p->g[i].end - p->g[i].first, splits = ceil_div(p->g[i].pages, p->split_pages);
    p->items += ceil_div((int)(n * rep), p->tile_rows) * splits;
    p->part_rows += n * n_heads * splits;
  }
  if (p->items * c->n_kv_heads > INT32_MAX) return fail(LNSKV_ERR_UNSUPPORTED, "too many row tiles");
  p->part_at = (std::max(p->ws_bytes, kWsHeaderBytes) + 255) & ~(size_t)255;
  p->ws_bytes = p->part_at + (size_t)p->part_rows * row;
  return LNSKV_OK;
}

}  // namespace
}  // namespace lnskv

using namespace lnskv;

extern "C" {

int lnskv_prefix_decode_workspace_size(const lnskv_pages* c, const int32_t* groups, int32_t n_groups, int32_t n_seq,
                                       int32_t n_heads, int32_t max_kv_len, size_t* bytes) {
  clear_error();
  if (!bytes) return fail(LNSKV_ERR_INVALID, "bytes is NULL");
  *bytes = 0;
  if (int rc = check_geometry(c)) return rc;
  if (int rc = check_var_shape(c, n_seq, n_heads, max_kv_len)) return rc;
  PrefixPlan p;
  if (int rc = plan_prefix(c, groups, n_groups, n_seq, n_heads, max_kv_len, &p)) return rc;
  *bytes = p.ws_bytes;
  return LNSKV_OK;
}

int lnskv_prefix_decode(const lnskv_pages* c, const float* q, float* out, const float* gate, const uint32_t* bt,
                        int32_t bt_stride, const int32_t* kv_len, const int32_t* groups, int32_t n_groups,
                        int32_t n_seq, int32_t n_heads, int32_t max_kv_len, float scale, void* ws, size_t ws_bytes,
                        lnskv_stream_t stream) {
  clear_error();
  if (int rc = check_var_call(c, q, out, bt, bt_stride, kv_len, n_seq, n_heads, max_kv_len, scale)) return rc;
  if (int rc = check_var_shape(c, n_seq, n_heads, max_kv_len)) return rc;
  PrefixPlan p;
  if (int rc = plan_prefix(c, groups, n_groups, n_seq, n_heads, max_kv_len, &p)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (int rc = var_workspace(&ws, ws_bytes, p.ws_bytes, st)) return rc;
  const DecodeArgs a = var_args(c, q, out, gate, bt, bt_stride, kv_len, n_heads, max_kv_len, scale, p.own, stream);
  const int d = (int)c->head_dim;
  uint8_t* base = static_cast<uint8_t*>(ws);
  OwnArgs o{};
  o.n_seq = n_seq;
  o.shares = p.shares;
  o.share_pages = p.share_pages;
  o.prefix.n_groups = p.n_groups;
  o.prefix.split_pages = p.split_pages;
  std::copy(p.g, p.g + p.n_groups, o.prefix.g);
  if (p.n_groups > 0) {
    PrefixArgs x{};
    x.pf.k_pages = a.k_pages;
    x.pf.v_pages = a.v_pages;
    x.pf.k_scales = a.k_scales;
    x.pf.v_scales = a.v_scales;
    x.pf.num_pages = c->num_pages;
    x.pf.n_kv = a.n_kv;
    x.k_pages = a.k_pages;
    x.v_pages = a.v_pages;
    x.k_scales = a.k_scales;
    x.v_scales = a.v_scales;
    x.q = q;
    x.bt = bt;
    x.kv_len = kv_len;
    x.part_acc = reinterpret_cast<float*>(base + p.part_at);
    x.part_ml = x.part_acc + (size_t)p.part_rows * d;
    x.bt_stride = bt_stride;
    x.n_kv = a.n_kv;
    x.n_heads = n_heads;
    x.rep = n_heads / a.n_kv;
    x.max_kv_len = max_kv_len;
    x.split_pages = p.split_pages;
    x.n_groups = p.n_groups;
    x.num_pages = c->num_pages;
    x.scale_log2 = a.scale_log2;
    std::copy(p.g, p.g + p.n_groups, x.g);
    o.prefix.part_acc = x.part_acc;
    o.prefix.part_ml = x.part_ml;
    const unsigned blocks = (unsigned)(p.items * a.n_kv);
    switch (c->dtype) {
      case LNSKV_DTYPE_F32: launch_prefix_f32<LNSKV_DTYPE_F32>(x, d, blocks, st); break;
      case LNSKV_DTYPE_F16:
        if (var_mfma(c)) launch_prefix_mfma<false>(x, d, p.tile_rows, blocks, st);
        else launch_prefix_f32<LNSKV_DTYPE_F16>(x, d, blocks, st);
        break;
      default:
        if (var_mfma(c)) launch_prefix_mfma<true>(x, d, p.tile_rows, blocks, st);
        else launch_prefix_f32<LNSKV_DTYPE_Q8A>(x, d, blocks, st);
        break;
    }
    if (int rc = hip_check("prefix kernel launch")) return rc;
  }
  if (p.shares == 0) return launch_generic<kPrefix>(c, a, p.own, n_seq, ws, o.prefix, st);
  if (p.shares > 1) {
    o.own_acc = reinterpret_cast<float*>(base + p.own_at);
    o.own_ml = o.own_acc + (size_t)p.shares * n_seq * n_heads * d;
  }
  const unsigned blocks = (unsigned)((int64_t)p.shares * n_seq * a.n_kv);
  const int rep = n_heads / a.n_kv;
  if (c->dtype == LNSKV_DTYPE_Q8A) {
    if (d == 256) launch_own_rep<true, 2>(a, o, rep, blocks, st);
    else launch_own_rep<true, 1>(a, o, rep, blocks, st);
  } else {
    if (d == 256) launch_own_rep<false, 2>(a, o, rep, blocks, st);
    else launch_own_rep<false, 1>(a, o, rep, blocks, st);
  }
  if (int rc = hip_check("own pages kernel launch")) return rc;
  if (p.shares > 1) {
    const unsigned jb = (unsigned)(((int64_t)n_seq * n_heads + kWavesPerBlock - 1) / kWavesPerBlock);
    if (d == 256) prefix_join_kernel<256><<<jb, kBlock, 0, st>>>(a, o);
    else prefix_join_kernel<128><<<jb, kBlock, 0, st>>>(a, o);
    return hip_check("prefix join kernel launch");
  }
  return LNSKV_OK;
}

}  // extern "C"
