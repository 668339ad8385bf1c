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
// 2. own kernel (f16 and Q8A pages, 128- and 256-wide heads; the tile kernel's
//    kernel elsewhere): work item = (sequence, kv head, share of its own pages);
//    a sequence with one share merges the prefix's rows and writes its output.
// 3. join kernel, where sequences may have several shares: their rows and the
//    prefix's into the output.
// Small calls leave out step 1: each sequence reads its group's pages itself.
#include "lnskv_decode_block.h"
#include "lnskv_decode_var.h"
#include "lnskv_prefill.h"

namespace lnskv {
namespace {

// Fewest pages of a split.  Us with 2 | 4 | 8, shared tokens x rows x kv heads: 547 x 164
// x 8 22.0 | 21.5 | 23.8, 193 x 12 x 4 (256-wide) 26.1 | 27.5 | 31.5, 63 x 16 x 8 12.5 |
// 13.4 | 13.4; tile kernel 503 x 8 x 8 21.7 | 24.0 | 29.0, 505 x 10 x 8 10.6 | 12.6 | 16.9.
constexpr int kSplitPages = 2;
// Splits of 128-row tiles from which tiles of 256 rows read each operand from LDS for
// twice the products.  Us, 128 | 256 rows, 512 rows x 8 kv heads, f16 pages: 4000 tokens
// (splits of 32 pages) 42.9 | 45.3, 8000 66.2 | 62.6, 16000 109 | 100; Q8A 51.3 | 50.8,
// 78.2 | 70.9, 125 | 111.
constexpr int kWidePages = 48;
// A sequence's own pages: shares of at most kSharePages pages (four waves, 16 each).
// Batches that leave compute units idle take smaller ones, but for short ones
// (kShareWhole pages), where the rows' way through memory and the join cost more: 48 x 4
// kv heads of up to 300 tokens, Q8A, 256-wide, in all 44.5 us whole and 54.8 in shares of
// kShareMin; 4 x 8 of up to 1000 tokens, f16, 21.0 in shares and 24.3 whole.  kSharePages
// 32 | 64 | 128, 64 x 8 of up to 4000 tokens: 165 | 165 | 171 us.  kShareMin 4 | 8 | 16, 4
// x 8 of up to 1000: 23.0 | 21.0 | 21.5.
constexpr int kSharePages = 64;
constexpr int kShareMin = 8;
constexpr int kShareWhole = 32;
// Small calls skip the prefix kernel: every sequence reads its group's pages itself, from
// L2 mostly.  On the matrix cores sequences of at most kDirectPages pages (one share, one
// launch), kDirectBytes of K and V in all with shared pages counted every time, and longer
// ones of at most kDirectLong pages of 128 elements in all (shares and their join).  Us,
// that | prefix and own pages apart, sequences x kv heads of pages: f16 128-wide 4 x 8 of 13
// 7.3 | 13.8, 16 x 8 of 57 13.3 | 19.2, 64 x 8 of 57 (228 MB) 22.3 | 26.4, 128 x 8 of 57
// (456 MB) 42.6 | 39.9; Q8A 128 x 8 of 57 (228 MB) 39.4 | 36.7, 256-wide 64 x 4 of 26 17.4 |
// 26.6; longer, f16 128-wide 2 x 8 of 82 11.4 | 17.1, 5 x 8 of 163 15.3 | 22.1, 5 x 8 of 257
// 22.2 | 20.2, 12 x 8 of 82 20.4 | 18.7, 12 x 4 of 82 19.2 | 25.4, 12 x 8 of 257 29.9 | 20.9;
// Q8A 5 x 4 of 163 14.2 | 24.6, 256-wide 5 x 4 of 163 26.9 | 34.1, 12 x 4 of 257 47 | 34.
// On the tile kernel kDirectUnits x (7 + heads per kv head) pages of 64 elements (a wave's
// products cost the same for one head and for 16, so what the prefix kernel saves by tiles
// of 16 rows falls with the heads): f32, 8 heads on one, 2 x 4 of 588 14 | 56, 6 x 4 of 588
// 24 | 41, 20 x 4 of 194 25.9 | 25.6, 60 x 4 of 88 32 | 27, 128-wide 60 x 4 of 32 19 | 25, 20
// x 4 of 194 47 | 36; 2 heads, 128-wide 6 x 8 of 88 16 | 22, 20 x 8 of 32 19.9 | 17.6; f16,
// 64-wide, 8 heads 6 x 4 of 588 19 | 36, 1 head 6 x 8 of 88 9.6 | 13.8.
constexpr int kDirectPages = 64;
constexpr int64_t kDirectBytes = (int64_t)192 << 20;
constexpr int64_t kDirectLong = 10240;
constexpr int64_t kDirectUnits = 1024;

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
// f32 pages, and 64-wide heads on every page type (lnskv_decode_tile.h): a
// wave per item of 16 rows and one split.  The waves of a block take the tiles of
// one split, or consecutive splits of few rows, and share nothing but the cache.
// Bound by the products (v_mfma_f32_16x16x4_f32, 32 cycles) once groups are large: 109
// sequences x 2 heads on 8 of 128 behind 4407 tokens, f32, 59 us in all (28 at the
// library's f32 rate), 68 with the page shared by four waves in LDS; by latency where they
// are small: 2 sequences x 8 heads on 4 of 64 behind 256 tokens 6.3 us.
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void prefix_tile_kernel(PrefixArgs a) {
  const int kvh = (int)(blockIdx.x % (unsigned)a.n_kv);
  const int wi = (int)(threadIdx.x / kWave), lane = (int)(threadIdx.x % kWave), g = lane >> 4, n = lane & 15;
  const PrefixItem it = prefix_item(
      a, __builtin_amdgcn_readfirstlane((int)(blockIdx.x / (unsigned)a.n_kv) * kWavesPerBlock + wi), 16);
  if (it.group < 0) return;  // wave-uniform; the waves share nothing
  const PrefixGroup gr = a.g[it.group];
  const int rows = (gr.end - gr.first) * a.rep, r0 = 16 * it.tile;
  const int rn = min(r0 + n, rows - 1);  // past the last row: that row again, never written
  const int sn = gr.first + rn / a.rep, hn = kvh * a.rep + rn % a.rep;
  const int limit = row_tokens(a, sn, gr.pages);
  int most = limit, least = limit;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    most = max(most, __shfl_xor(most, o, kWave));
    least = min(least, __shfl_xor(least, o, kWave));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  const int pg0 = it.split * a.split_pages;
  const int pg1 = min(min(gr.pages, pg0 + a.split_pages), (most + kPage - 1) / kPage);
  const uint32_t* bt_row = a.bt + (size_t)gr.first * a.bt_stride;
  TileState<DT, D> st;
  tile_init<DT, D>(st, a.q + ((size_t)sn * a.n_heads + hn) * D, a.scale_log2, g);
  for (int p = pg0; p < pg1; p += kWave) {  // 64 table entries at a time
    const uint32_t btv = p + lane < a.bt_stride ? bt_row[p + lane] : 0xFFFFFFFFu;
    tile_pages<DT, D>(
        a, kvh, g, n, 0, 1, min(pg1 - p, kWave), [&](int i) { return __builtin_amdgcn_readlane(btv, i); },
        [&](int i, bool valid, TilePage<DT, D>& pg) {
          const int tok0 = (p + i) * kPage;
          tile_consume<DT, D>(
              st, pg, valid && tok0 + kPage <= least, g, [&](int t) { return valid && tok0 + t < limit; },
              [&](int t) { return valid && tok0 + t < most; });
        });
  }
  st.l = sum_xor16(sum_xor32(st.l));
  if (lane < 16 && r0 + n < rows) {
    const RowOut o = row_out<D>(a, it, sn, hn);
    o.ml[0] = st.m;
    o.ml[1] = st.l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * g + i;
    if (r < rows) {
      const RowOut o = row_out<D>(a, it, gr.first + r / a.rep, kvh * a.rep + r % a.rep);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<float4v*>(o.acc + 64 * c + 4 * n) =
            tile_out<DT, D>(st, c, i);
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
// Bound by its chain of LDS reads, products and softmax per pair of pages, two waves to a
// SIMD; short splits by latency and the partial rows' bytes.  128 sequences x 4 heads on 8
// behind 16384 tokens, f16: 85 to 89 us (34 GFLOP, twice that in products of hi and lo
// parts: 59 us at the rate of a large library product); 3 x 16 sequences x 4 heads on 4 of
// 256 behind 4090 tokens, Q8A: 26 us; 32 x 4 on 8 behind 2048, f16: 12.6 us.
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
// merge them head by head.  No workgroup depends on another.  Bound by HBM in large
// batches: 128 sequences x 8 kv heads of 64 to 1024 tokens, f16, with the prefix's 16
// partial rows per head: 84 us (318 MB: 66 at a large copy's rate; three waves to a SIMD
// instead of two spill and take 94); 32 of up to 512 12 to 15.
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
  o.p0 = x.prefix.split_pages > 0 ? min(o.prefix.pages * kPage, o.L) : 0;
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

template <int REP, bool Q8, int NH>
__global__ __launch_bounds__(kWave* kBlockWaves) __attribute__((amdgpu_waves_per_eu(NH == 1 ? 2 : 1)))
void prefix_own_kernel(DecodeArgs a, OwnArgs x) {
  constexpr int NW = kBlockWaves, D = NH * kD, C = D / kWave;
  __shared__ BlockLds<REP, Q8, NH> sm;
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
    PieceLoads<REP, NH> pl;
    piece_loads<REP, false, false, Q8, NH>(a, s, kvh, o.p0 / kPage + i0, pl);
    if (x.prefix.split_pages == 0) {  // shared pages too: fewer than the window's 64 entries a wave
      const int e = i0 + lane;
      if (e < a.bt_stride && e < o.prefix.pages) pl.btv = a.bt[(size_t)o.prefix.first * a.bt_stride + e];
    }
    block_piece<REP, Q8, NH>(a, sm, wi, s, kvh, pl, o.p0 / kPage, i0, i1, o.L);
  }
  __syncthreads();
  const int nw = hi > lo ? ceil_div(hi - lo, per) : 0;  // waves that left rows
  for (int h = wi; h < REP; h += NW) {  // wave-uniform
    const size_t hrow = (size_t)s * a.n_heads + (size_t)kvh * REP + h;
    float M, Ls, A[C];
    block_merge<REP, Q8, NH>(sm, nw, h, M, Ls, A);
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
    case 1: prefix_own_kernel<1, Q8, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x); break;
    case 2: prefix_own_kernel<2, Q8, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x); break;
    case 4: prefix_own_kernel<4, Q8, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x); break;
    default: prefix_own_kernel<8, Q8, NH><<<blocks, kWave * kBlockWaves, 0, st>>>(a, x); break;
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
void launch_prefix_tile(const PrefixArgs& a, int d, int64_t items, hipStream_t st) {
  const unsigned blocks = (unsigned)((items + kWavesPerBlock - 1) / kWavesPerBlock * a.n_kv);
  if (d == 64) prefix_tile_kernel<DT, 64><<<blocks, kBlock, 0, st>>>(a);
  if constexpr (DT == LNSKV_DTYPE_F32) {
    if (d == 128) prefix_tile_kernel<DT, 128><<<blocks, kBlock, 0, st>>>(a);
    if (d == 256) prefix_tile_kernel<DT, 256><<<blocks, kBlock, 0, st>>>(a);
  }
}

// ---------------------------------------------------------------------------
// The host's view of a call.
struct PrefixPlan {
  bool direct = false;    // every sequence reads the shared pages itself
  VarPlan own;            // the tile kernel over the sequences' own pages
  int shares = 0;         // own kernel: shares of a sequence at most (0: the tile kernel)
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
  const int64_t all = (int64_t)max_kv_len / kPage + 1;
  int64_t own_pages = 0, most = 0, tiles = 0, wide = 0, max_shared = 0;  // summed over sequences; of one sequence
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
    tiles += ceil_div(n * rep, var_mfma(c) ? 128 : 16);
    wide += ceil_div(n * rep, 256);
    max_shared = std::max(max_shared, shared);
  }
  if (at < n_seq) most = all;
  own_pages += (n_seq - at) * all;
  const size_t row = ((size_t)d + 2) * sizeof(float);
  if (schedule_setting() == kScheduleAuto) {
    const int64_t units = all * n_seq * c->n_kv_heads;
    const int64_t page = kPage * 2 * d * (c->dtype == LNSKV_DTYPE_F16 ? 2 : 1);
    p->direct = !var_mfma(c)           ? units * (d / 64) <= kDirectUnits * (7 + rep)
                : all <= kDirectPages ? units <= kDirectBytes / page
                                      : units * (d / 128) <= kDirectLong;
    if (p->direct) {
      own_pages = all * n_seq;
      most = all;
    }
  }
  if (var_mfma(c)) {
    // shares of at most kSharePages pages, fewer where that leaves compute units idle
    const int64_t units = own_pages * c->n_kv_heads;
    p->share_pages = n_seq * (int64_t)c->n_kv_heads >= 256 || most <= (p->direct ? kDirectPages : kShareWhole)
                         ? kSharePages
                         : (int)std::min<int64_t>(kSharePages, std::max<int64_t>(kShareMin, (units + 511) / 512));
    p->shares = (int)std::max<int64_t>(1, (most + p->share_pages - 1) / p->share_pages);
    if ((int64_t)p->shares * n_seq * c->n_kv_heads > INT32_MAX)
      return fail(LNSKV_ERR_UNSUPPORTED, "a batch of more than 2^31 shares");
    p->own_at = kWsHeaderBytes;
    p->ws_bytes = p->shares > 1 ? kWsHeaderBytes + (size_t)p->shares * n_seq * n_heads * row : 0;
  } else {
    if (int rc = plan_tiles(c, n_seq, n_heads, most, &p->own)) return rc;
    p->ws_bytes = p->own.ws_bytes;
  }
  if (p->n_groups == 0 || p->direct) return LNSKV_OK;
  // splits of equal pages: as many items as the card takes at once (a workgroup of
  // the matrix-core kernel per compute unit; of the tile kernel's waves two per SIMD
  // with 64-wide heads, else one)
  const int64_t fill = var_mfma(c) ? 256 : d == 64 ? 2048 : 1024;
  auto split_pages = [&](int64_t t) {
    const int64_t want = std::max<int64_t>(1, fill / (t * c->n_kv_heads));
    return (int)std::max<int64_t>(kSplitPages, (max_shared + want - 1) / want);
  };
  // matrix-core kernel: tiles of 256 rows (two heads of a sequence per column) where
  // splits are long and none of these tiles is half empty
  p->tile_rows = !var_mfma(c) ? 16 : d == 128 && rep > 1 && 2 * wide == tiles && split_pages(tiles) >= kWidePages ? 256 : 128;
  p->split_pages = split_pages(p->tile_rows == 256 ? wide : tiles);
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
  if (p.n_groups > 0 && var_mfma(c) && c->dtype == LNSKV_DTYPE_Q8A &&
      (uint64_t)c->num_pages * kPage * c->n_kv_heads * sizeof(float) > 0x7FFFFFF0u)  // the page pipeline's scale offsets
    return fail(LNSKV_ERR_UNSUPPORTED, "shared prefixes on Q8A pages need scale arrays under 2 GiB (%u pages x %u kv heads)",
                c->num_pages, c->n_kv_heads);
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
  o.prefix.split_pages = p.direct ? 0 : p.split_pages;
  std::copy(p.g, p.g + p.n_groups, o.prefix.g);
  if (p.n_groups > 0 && !p.direct) {
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
      case LNSKV_DTYPE_F32: launch_prefix_tile<LNSKV_DTYPE_F32>(x, d, p.items, st); break;
      case LNSKV_DTYPE_F16:
        if (var_mfma(c)) launch_prefix_mfma<false>(x, d, p.tile_rows, blocks, st);
        else launch_prefix_tile<LNSKV_DTYPE_F16>(x, d, p.items, st);
        break;
      default:
        if (var_mfma(c)) launch_prefix_mfma<true>(x, d, p.tile_rows, blocks, st);
        else launch_prefix_tile<LNSKV_DTYPE_Q8A>(x, d, p.items, st);
        break;
    }
    if (int rc = hip_check("prefix kernel launch")) return rc;
  }
  if (p.shares == 0) return launch_tiles<kPrefix>(c, a, p.own, n_seq, ws, o.prefix, st);
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
