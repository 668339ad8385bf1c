// A workgroup per (sequence, kv head) for the decode variants on f16 and Q8A pages
// with 128- or 256-wide heads: its waves take consecutive pages and their rows
// merge in LDS, with no workspace and no other workgroup to wait for.
#pragma once

#include "lnskv_decode_mfma.h"

namespace lnskv {
namespace {

constexpr int kBlockWaves = 4;

template <int REP, bool Q8, int NH>
struct BlockLds {
  static constexpr int kSlots = Q8 ? 1 : 2;
  static constexpr int kRow = NH * kD + 2;  // an LDS partial row: acc, m, l
  __attribute__((aligned(16))) uint8_t vring[kBlockWaves][kSlots * NH * kVSlot];
  __attribute__((aligned(16))) float part[kBlockWaves * REP * kRow];
};

// Wave wi's row of partial results of pages [i0, i1), counted from page pg0; tokens
// from L on are masked (kSink: what the span does not see).  pl: piece_loads of the
// first of them.
template <int REP, bool Q8, int NH, int VAR = kPlain, class... SP>
__device__ __forceinline__ void block_piece(const DecodeArgs& a, BlockLds<REP, Q8, NH>& sm, int wi, int s, int kvh,
                                            PieceLoads<REP, NH>& pl, int pg0, int i0, int i1, int L, const SP&... sp) {
  PieceOut po;
  po.final = false;
  po.pbase = (size_t)wi * REP;
  po.pstride = 1;
  po.in_lds = true;
  po.lds = (__attribute__((address_space(3))) float*)sm.part;
  lds_u8* ring = (lds_u8*)sm.vring[wi];
  const int ta = (pg0 + i0) * kPage, tb = VAR == kSink ? (pg0 + i1) * kPage : min(L, (pg0 + i1) * kPage);
  if constexpr (Q8)
    run_piece_q8<REP, 2, false, NH, false, VAR>(a, ring, ring, pl, true, s, kvh, ta, tb, false, L - 1, po, nullptr, sp...);
  else
    run_piece<REP, false, 2, false, NH, VAR>(a, ring, ring, pl, true, s, kvh, ta, tb, false, L - 1, po, nullptr, sp...);
}

// Head h's rows of the first nw waves; lane l holds columns l + 64 c.
template <int REP, bool Q8, int NH>
__device__ __forceinline__ void block_merge(const BlockLds<REP, Q8, NH>& sm, int nw, int h, float& M, float& Ls,
                                            float (&A)[2 * NH]) {
  using Lds = BlockLds<REP, Q8, NH>;
  constexpr int D = NH * kD;
  const int lane = (int)(threadIdx.x % kWave);
  M = kMInit;
  Ls = 0.0f;
#pragma unroll
  for (int c = 0; c < 2 * NH; ++c) A[c] = 0.0f;
  for (int w = 0; w < nw; ++w) {
    const float* row = sm.part + ((size_t)w * REP + h) * Lds::kRow;
    const float m = row[D], Mn = fmaxf(M, m);
    const float wa = fast_exp2(M - Mn), wb = fast_exp2(m - Mn);
    Ls = Ls * wa + row[D + 1] * wb;
#pragma unroll
    for (int c = 0; c < 2 * NH; ++c) A[c] = A[c] * wa + row[lane + c * kWave] * wb;
    M = Mn;
  }
}

}  // namespace
}  // namespace lnskv
