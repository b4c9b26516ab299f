// Products of a few rows an expert with 4-bit weights.
//
// A wave has WT tiles of features (with a second matrix WT / 2 of each) and up to sixteen rows; WK waves of a workgroup share the columns, a tile of 128 in
// turn each, and their sums are added up in the LDS, in order.  A word's codes become 16 + q in the activations' type by a shift and a mask-and-or for two
// of them (bf16: the mantissa's upper four bits are its bits 3 - 6, fp16: 6 - 9); the products with a column of ones are the sums of the rows' group,
//   sum x scale (q - zero) = scale (sum x (16 + q) - (16 + zero) sum x)
// in fp32, where 16 + q costs four bits of 24 of which 16-bit activations have eleven.
//
// What bounds it: reading the weights.  A kernel that only reads as much takes 18.6 us for the 118 MiB of one token (top-2 of 8 gated experts of [4096,
// 14336]), 73 for the 472 MiB of all eight, this one 25 and 82.  Many waves with one block each under way read faster than fewer with several (one token
// 25 us; two blocks 28.8, four, of fewer waves, 33.4), and rows that are not there are not read: 64 lanes of x are as long in the load unit as the weights.
#include "gmm_4bit.h"

namespace mbx {
namespace {

constexpr int rows_waves(int wk) { return wk > 4 ? wk : 4; }   // of a workgroup

template <int DT, int WT, bool TWO, int GROUP, int WK>
__global__ void __launch_bounds__(rows_waves(WK) * kWave, 4)
rows_4bit_kernel(const Rows4bit g) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32, kWaves = rows_waves(WK), WF = kWaves / WK;
  constexpr int kFeatureTiles = TWO ? WT / 2 : WT;
  __shared__ float sums[kWaves][WT * 4][kWave];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), f = lane % 16, part = lane / 16;
  const int wk = wave % WK, wf = wave / WK;
  int expert, first, end;
  if (!find_rows(g, 16, expert, first, end)) return;   // alike for all waves: none is left at the barrier
  const int tiles = (g.n + 15) / 16, blocks = (g.k + 127) / 128, tile0 = ((int)blockIdx.x * WF + wf) * kFeatureTiles;
  const Weights4bit<DT, WT, TWO, GROUP> weights(g, expert, tile0, tiles, blocks);
  typename Weights4bit<DT, WT, TWO, GROUP>::Block now;
  if (wk < blocks) weights.template fetch<true>(now, wk);    // on its way before the rows are looked up
  const bool live = first + f < end;                         // lanes of other rows read nothing and stay zero
  const uint16_t* const row = row_of(g, live ? first + f : end - 1);
  u32x4_t x[4] = {};
  f32x4_t y[WT] = {};
  const u32x4_t ones = ones_of<DT>();
  const CodeBits<DT> codes;
  for (int b = wk; b < blocks; b += WK) {
    const int c0 = b * kTileColumns + 8 * part;
    if (live) {
      if ((b + 1) * kTileColumns <= g.k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_memcpy(&x[j], row + c0 + 32 * j, 16);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) read_columns(row, c0 + 32 * j, g.k, x[j]);
      }
    }
    uint32_t scale[WT][kGroups], off[WT][kGroups];
    const uint32_t scale_mask = weights.mask_of(b);
#pragma unroll
    for (int t = 0; t < WT; ++t) weights.scales(now, t, scale_mask, scale[t], off[t]);
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      f32x4_t of_ones = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = q * kEach; j < (q + 1) * kEach; ++j) of_ones = mfma_16x16x32<DT>(x[j], ones, of_ones);
#pragma unroll
      for (int t = 0; t < WT; ++t) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = q * kEach; j < (q + 1) * kEach; ++j) acc = mfma_16x16x32<DT>(x[j], sixteen_and<DT>(now.words[t][j], codes.mask, codes.bits), acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[t][i] = fmaf(__uint_as_float(scale[t][q]), fmaf(__uint_as_float(off[t][q]), of_ones[i], acc[i]), y[t][i]);
      }
      // a group's sums before the next group's products: all products first take more registers than there are
#pragma unroll
      for (int t = 0; t < WT; ++t) asm volatile("" : "+v"(y[t]));
      if constexpr (kGroups > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (b + WK < blocks) weights.template fetch<true>(now, b + WK);
  }
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][t * 4 + i][lane] = y[t][i];
  __syncthreads();
  // lane l, place i of a tile: row 4 (l / 16) + i, feature l % 16
  for (int v = wk; v < kFeatureTiles * 4; v += WK) {
    const int t = v / 4, i = v % 4;
    const auto sum = [&](int tile) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) s += sums[wf * WK + w][tile * 4 + i][lane];
      return s;
    };
    const int r = first + 4 * part + i, feature = (tile0 + t) * 16 + f;
    if (r >= end || feature >= g.n) continue;
    float c = sum(TWO ? 2 * t : t);
    if (g.act >= 0) c = activated(c, g.act);
    if constexpr (TWO) c *= sum(2 * t + 1);
    ((E*)g.c)[(int64_t)r * g.n + feature] = Elem<DT>::from_f32(c);
  }
}

template <int DT, int WT, bool TWO, int GROUP, int WK>
void launch(const Rows4bit& g, int64_t slots, hipStream_t s) {
  const int64_t waves = pieces_of(g.n, 16 * (TWO ? WT / 2 : WT));
  for_slots(g, slots, [=](const Rows4bit& of, unsigned tiles) {
    rows_4bit_kernel<DT, WT, TWO, GROUP, WK><<<dim3((unsigned)pieces_of(waves, rows_waves(WK) / WK), tiles), rows_waves(WK) * kWave, 0, s>>>(of);
  });
}

// More tiles a wave share a reading of the rows, fewer leave more waves; the more waves share the columns the shorter the way of each.  By the tiles that
// the experts with rows have (us; tiles a wave / waves that share the columns):
//     256 (one expert of [4096, 4096], a row)             1/8 5.5, 2/8 6.4, 4/8 30
//     512 (2 of [14336, 4096], a row each)                1/8 19.4, 2/8 16.5, 1/4 23.9
//    1056 (6 gated ones of [2048, 1408], a row each)      2/8 7.9, 2/4 8.0, 4/8 8.8, 4/4 9.6
//    2048 (8 of [14336, 4096], 4 rows each)               4/8 43.7, 2/8 46.7, 2/4 47.5, 4/4 52.6
//    3584 (2 gated ones of [4096, 14336], a row each)     4/4 25.0, 2/8 25.4, 2/4 25.9, 4/8 26.4
//    5280 (30 gated ones of [2048, 1408], a row each)     2/4 20.0, 4/4 20.6, 4/8 21.5
//   14336 (8 gated ones of [4096, 14336], 4 rows each)    4/4 82, 4/2 87, 2/4 91, 4/8 91
template <int DT, bool TWO, int GROUP>
void choose(const Rows4bit& g, int64_t slots, int64_t experts, hipStream_t s) {
  const int64_t tiles = pieces_of(g.n, 16) * (TWO ? 2 : 1) * experts;
  if (tiles <= 400 && !TWO) launch<DT, TWO ? 2 : 1, TWO, GROUP, 8>(g, slots, s);
  else if (tiles <= 1536) launch<DT, 2, TWO, GROUP, 8>(g, slots, s);
  else if (tiles <= 2816) launch<DT, 4, TWO, GROUP, 8>(g, slots, s);
  else launch<DT, 4, TWO, GROUP, 4>(g, slots, s);
}

template <int DT, bool TWO>
void by_group(const Rows4bit& g, int group, int64_t slots, int64_t experts, hipStream_t s) {
  if (group == 32) choose<DT, TWO, 32>(g, slots, experts, s);
  else if (group == 64) choose<DT, TWO, 64>(g, slots, experts, s);
  else choose<DT, TWO, 128>(g, slots, experts, s);
}

}  // namespace

int launch_rows_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, int64_t experts, hipStream_t s) {
  const bool two = g.b[1].words != nullptr;
  if (dtype == MBX_BF16) two ? by_group<MBX_BF16, true>(g, group, slots, experts, s) : by_group<MBX_BF16, false>(g, group, slots, experts, s);
  else two ? by_group<MBX_F16, true>(g, group, slots, experts, s) : by_group<MBX_F16, false>(g, group, slots, experts, s);
  return launch_status();
}

}  // namespace mbx
