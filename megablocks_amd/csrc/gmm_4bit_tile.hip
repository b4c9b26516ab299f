// Products of some dozens of rows an expert with 4-bit weights.
//
// A workgroup has 32 rows and each of its four waves WT tiles of features of its own (with a second matrix WT / 2 of each), all columns.  The rows' columns
// are fetched three blocks of 128 ahead and shared through the LDS: 256 bytes a row, its 16-byte pieces in the order piece ^ row, so that the 16 rows of a
// read are 16 different bank groups.  The weights go from memory to the operands as in gmm_4bit_rows.hip, each wave's own.  What 16 + q is off by is taken off
// at the start: sums of the next block's rows, made by two of the waves, are what its products are added to.
//
// What bounds it: the instructions that make operands of the codes, two for two weights, as many as the matrix instructions can hide or more, and a barrier a
// block.  Us (and TFLOP/s) of the first products of 8 gated experts of [4096, 14336], by rows an expert: 16: 100, 32: 131 (460), 64: 230 (522), 96: 305;
// 128: 381, 256: 698 (689).  With the sums made by every wave for itself, 40 matrix instructions a block in place of 32: 150 (32 rows), 469 (128).
#include "gmm_4bit.h"

namespace mbx {
namespace {

constexpr int kRowTiles = 2;   // of 16

template <int DT, int WT, bool TWO, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(4 * kWave, WT == 2 ? 4 : 2)
tile_4bit_kernel(const Rows4bit g) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32, MT = kRowTiles;
  constexpr int kFeatureTiles = TWO ? WT / 2 : WT;
  __shared__ u32x4_t staged[3][16 * MT][16];
  __shared__ f32x4_t sums[2][kGroups][4 * MT];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), f = lane % 16, part = lane / 16;
  int expert, first, end;
  if (!find_rows(g, 16 * MT, expert, first, end)) return;   // alike for all waves: none is left at a barrier
  const int tiles = (g.n + 15) / 16, blocks = (g.k + 127) / 128, tile0 = ((int)blockIdx.x * 4 + wave) * kFeatureTiles;
  const Weights4bit<DT, WT, TWO, GROUP> weights(g, expert, tile0, tiles, blocks);
  typename Weights4bit<DT, WT, TWO, GROUP>::Block next;
  // thread i stages piece i % 16 of rows i / 16, i / 16 + 16, ...; rows past the last are the last again
  const int piece = (int)threadIdx.x % 16, stage_row = (int)threadIdx.x / 16;
  const uint16_t* row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + stage_row;
    row[m] = row_of(g, r < end ? r : end - 1);
  }
  u32x4_t x_next[MT];
  const auto fetch_rows = [&](int b) {
#pragma unroll
    for (int m = 0; m < MT; ++m) read_columns(row[m], b * kTileColumns + 8 * piece, g.k, x_next[m]);
  };
  const auto stage = [&](int buffer) {
#pragma unroll
    for (int m = 0; m < MT; ++m) staged[buffer][16 * m + stage_row][piece ^ stage_row] = x_next[m];
  };
  // Sums of the rows' columns of each group, a wave a tile of rows; without zeros times -24, which is what a code of 0 is off by
  const u32x4_t ones = ZEROS ? ones_of<DT>() : all_of<DT>(-24.f);
  const auto sum_up = [&](int buffer, int to) {
    if (wave >= MT) return;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      f32x4_t sum = {};
#pragma unroll
      for (int j = q * kEach; j < (q + 1) * kEach; ++j) sum = mfma_16x16x32<DT>(staged[buffer][16 * wave + f][(4 * j + part) ^ f], ones, sum);
      if (f == 0) sums[to][q][4 * wave + part] = sum;
    }
  };
  f32x4_t y[WT][MT] = {};
  const CodeBits<DT> codes;
  fetch_rows(0);
  weights.template fetch<false>(next, 0);
  stage(0);
  if (blocks > 1) {
    fetch_rows(1);
    stage(1);
  }
  if (blocks > 2) fetch_rows(2);
  __syncthreads();
  sum_up(0, 0);
  __builtin_amdgcn_s_waitcnt(0x0f70);     // all loads: the loop's waits are then for its own alone
  int buffer = 0;
  for (int b = 0; b < blocks; ++b) {
    const auto now = next;
    const int after = buffer == 2 ? 0 : buffer + 1;
    __syncthreads();       // the rows of blocks b and b + 1 and the sums of b are there, and what is of block b - 1 no longer read
    if (b + 1 < blocks) {
      if (b + 2 < blocks) stage(after == 2 ? 0 : after + 1);
      if (b + 3 < blocks) fetch_rows(b + 3);
      weights.template fetch<false>(next, b + 1);
      sum_up(after, (b + 1) & 1);
    }
    const u32x4_t(*const x_now)[16] = staged[buffer];
    uint32_t scale[WT][kGroups], off[WT][kGroups];
    const uint32_t scale_mask = weights.mask_of(b);
#pragma unroll
    for (int t = 0; t < WT; ++t) weights.scales(now, t, scale_mask, scale[t], off[t]);
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      f32x4_t acc[WT][MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const f32x4_t sum = sums[b & 1][q][4 * m + part];
#pragma unroll
        for (int t = 0; t < WT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][m][i] = ZEROS ? __uint_as_float(off[t][q]) * sum[i] : sum[i];
      }
#pragma unroll
      for (int j = q * kEach; j < (q + 1) * kEach; ++j) {
        u32x4_t x[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) x[m] = x_now[16 * m + f][(4 * j + part) ^ f];
#pragma unroll
        for (int t = 0; t < WT; ++t) {
          const u32x4_t w = sixteen_and<DT>(now.words[t][j], codes.mask, codes.bits);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[t][m] = mfma_16x16x32<DT>(x[m], w, acc[t][m]);
        }
      }
#pragma unroll
      for (int t = 0; t < WT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[t][m][i] = fmaf(__uint_as_float(scale[t][q]), acc[t][m][i], y[t][m][i]);
          asm volatile("" : "+v"(y[t][m]));   // a group's sums before the next group's products
        }
    }
    buffer = after;
  }
#pragma unroll
  for (int t = 0; t < kFeatureTiles; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = first + 16 * m + 4 * part + i, feature = (tile0 + t) * 16 + f;
        float c = y[TWO ? 2 * t : t][m][i];
        if (g.act >= 0) c = activated(c, g.act);
        if constexpr (TWO) c *= y[TWO ? 2 * t + 1 : t][m][i];
        if (r < end && feature < g.n) ((E*)g.c)[(int64_t)r * g.n + feature] = Elem<DT>::from_f32(c);
      }
}

template <int DT, int WT, bool TWO, int GROUP>
void launch(const Rows4bit& g, int64_t slots, hipStream_t s) {
  for_slots(g, slots, [=](const Rows4bit& of, unsigned tiles) {
    const dim3 grid((unsigned)pieces_of(g.n, 64 * (TWO ? WT / 2 : WT)), tiles);
    if (g.b[0].zeros) tile_4bit_kernel<DT, WT, TWO, GROUP, true><<<grid, 4 * kWave, 0, s>>>(of);
    else tile_4bit_kernel<DT, WT, TWO, GROUP, false><<<grid, 4 * kWave, 0, s>>>(of);
  });
}

// Four tiles a wave where that leaves six workgroups a compute unit (us, two / four: 8 gated experts of [4096, 14336], 16 rows, 1344 workgroups 110 / 120, 32 rows,
// 1792, 155 / 138 (each some 5 % shorter since); 64 of [2048, 1408], 31 rows, 1386: 64 / 63, 65 rows, 2134: 129 / 117; 8 of [14336, 4096] without a gate, 64 rows, 384: 143 / 170)
template <int DT, bool TWO, int GROUP>
void choose(const Rows4bit& g, int64_t slots, hipStream_t s) {
  if (pieces_of(g.n, 64 * (TWO ? 2 : 4)) * slots >= 1536) launch<DT, 4, TWO, GROUP>(g, slots, s);
  else launch<DT, 2, TWO, GROUP>(g, slots, s);
}

template <int DT, bool TWO>
void by_group(const Rows4bit& g, int group, int64_t slots, hipStream_t s) {
  if (group == 32) choose<DT, TWO, 32>(g, slots, s);
  else if (group == 64) choose<DT, TWO, 64>(g, slots, s);
  else choose<DT, TWO, 128>(g, slots, s);
}

}  // namespace

int launch_tiles_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, hipStream_t s) {
  const bool two = g.b[1].words != nullptr;
  if (dtype == MBX_BF16) two ? by_group<MBX_BF16, true>(g, group, slots, s) : by_group<MBX_BF16, false>(g, group, slots, s);
  else two ? by_group<MBX_F16, true>(g, group, slots, s) : by_group<MBX_F16, false>(g, group, slots, s);
  return launch_status();
}

}  // namespace mbx
