// Products of hundreds to thousands of rows an expert with 4-bit weights.
//
// A workgroup has 64 rows, four waves with 64 features each (with a second matrix 32 of each), all columns; rows, weights and the start of the sums as in
// gmm_4bit_tile.hip.  A wave goes over its block of 128 columns a unit at a time, a group of columns of one tile of features: 4 to 16 matrix instructions, and
// next to each, in this order, two instructions of making the next operand of codes and one or two that scale and add up the unit before.  The rows of a
// block are read from the LDS once, into the registers that the block before leaves with its last tile of features, and a tile's words are loaded
// where its last operand has been made, three quarters of a block ahead.  That is the 256 registers there are for two waves on a SIMD.
//
// What bounds it: a SIMD issues one vector instruction in 4 cycles, a matrix instruction of 16 x 16 x 32 takes two such places (measured: 16 cycles alone, 9 ns
// with three others, 12 ns with five): 70 of them and 297 others a block are 437 places, of which 80 % are used.  First products of 8 gated experts of
// [4096, 14336], 256 / 512 / 1024 rows an expert: 623 / 1121 / 2107 us (772 / 858 / 913 TFLOP/s); values made in 16 bits and multiplied by the grouped kernels
// 1380 / 1799 / 2016, each weight rounded on the way.  128 rows a workgroup and one wave a SIMD with all 512 registers: 2245, its instructions one after the other.
// Groups of 32, 512 rows of 8 experts of [14336, 4096]: 827 us (582 TFLOP/s): four times the sums.
#include "gmm_4bit.h"

namespace mbx {
namespace {

constexpr int kRowTiles = 4, kFeatureWaves = 4, kTiles = 4;   // 64 rows a workgroup; 4 waves of 4 tiles of features

template <int DT, bool TWO, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kFeatureWaves * kWave, 2)
long_4bit_kernel(const Rows4bit g) {
  typedef typename Elem<DT>::type E;
  constexpr int MT = kRowTiles, WT = kTiles, kGroups = 128 / GROUP, kEach = GROUP / 32, kFlush = 8 / kEach;
  constexpr int kFeatureTiles = TWO ? WT / 2 : WT;
  static_assert(MT == kFeatureWaves && WT == 4, "a wave sums up a tile of rows, a quarter of the columns with each tile of features");
  __shared__ u32x4_t staged[3][16 * MT][16];
  __shared__ f32x4_t sums[2][kGroups][4 * MT];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), f = lane % 16, part = lane / 16;
  int expert, first, end;
  if (!find_rows(g, 16 * MT, expert, first, end)) return;   // alike for all waves: none is left at a barrier
  const int tiles = (g.n + 15) / 16, blocks = (g.k + 127) / 128, tile0 = ((int)blockIdx.x * kFeatureWaves + wave) * kFeatureTiles;
  typedef Weights4bit<DT, WT, TWO, GROUP> Weights;
  const Weights weights(g, expert, tile0, tiles, blocks);
  typename Weights::Block now;
  // thread i stages piece i % 16 of rows i / 16, i / 16 + 16, ...; rows past the last are the last again
  const int piece = (int)threadIdx.x % 16, stage_row = (int)threadIdx.x / 16;
  const uint16_t* row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + stage_row;
    row[m] = row_of(g, r < end ? r : end - 1) + (8 * piece < g.k ? 8 * piece : 0);
  }
  u32x4_t x_next[MT];
  const auto fetch_rows = [&](int b) {
    const int c = b * kTileColumns < g.k - 8 * piece ? b * kTileColumns : 0;     // rows are whole pieces: past the last, the first
#pragma unroll
    for (int m = 0; m < MT; ++m) __builtin_memcpy(&x_next[m], row[m] + c, 16);
  };
  const auto stage = [&](int buffer, int b) {
    if (b + 1 == blocks && b * kTileColumns + 8 * piece >= g.k) {
#pragma unroll
      for (int m = 0; m < MT; ++m) x_next[m] = u32x4_t{};
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) staged[buffer][16 * m + stage_row][piece ^ stage_row] = x_next[m];
  };
  const auto ones = [] {      // made where they are used: registers are short
    uint32_t one = all_of<DT>(ZEROS ? 1.f : -24.f)[0];
    asm volatile("" : "+v"(one));
    return u32x4_t{one, one, one, one};
  };
  const CodeBits<DT> codes;

  u32x4_t x[kEach][MT];       // the rows of a group
  const auto read_x = [&](int buffer, int j, u32x4_t (&to)[MT]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) to[m] = staged[buffer][16 * m + f][(4 * j + part) ^ f];
  };

  fetch_rows(0);
  // what the call has checked has checked: a tile's words and scales are less than 2^32 bytes
  const auto fetch_words = [&](int t, int b) { now.words[t] = load_at<u32x4_t>(weights.words_at[t], 0, (uint32_t)b * (kTileWords * 4) + weights.word_lane); };
  // The pieces of 4 bytes with the lane's scales, one load whatever the type; as 16 bits the lane's half is shifted up and the other cut off
  const int scale_shift = weights.wide ? 2 : 1;
  const uint32_t scale_at = weights.scale_lane << scale_shift & ~3u, half_up = weights.wide || lane % 2 ? 0 : 16, half_mask = weights.wide ? ~0u : 0xffff0000u;
  const auto fetch_scales = [&](int b) {
    const uint32_t block = (uint32_t)b * (kGroups * 16);
#pragma unroll
    for (int t = 0; t < WT; ++t) now.scale[t] = load_at<uint32_t>(weights.scales_at[t], 0, (block << scale_shift) + scale_at);
    if constexpr (ZEROS) {
#pragma unroll
      for (int t = 0; t < WT; ++t) now.zero[t] = load_at<uint8_t>(weights.zeros_at[t], 0, block + weights.scale_lane);
    }
  };
  const auto scales = [&](int t, uint32_t (&scale)[kGroups], uint32_t (&off)[kGroups]) {
    const uint32_t raw = (now.scale[t] << half_up) & half_mask;
    float s = __uint_as_float(raw);
    if constexpr (DT == MBX_F16) s = weights.wide ? s : Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(raw >> 16)));
    spread<kGroups>(__float_as_uint(s), scale);
    if constexpr (ZEROS) spread<kGroups>(__float_as_uint(-16.f - (float)now.zero[t]), off);
  };
  stage(0, 0);
  fetch_rows(1);
  stage(1, 1);
  fetch_rows(2);
  // after the rows, as in the loop: the first use of the words is behind all loads so far, and a wait in the loop for the loop's own alone
  fetch_scales(0);
#pragma unroll
  for (int t = 0; t < WT; ++t) fetch_words(t, 0);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    f32x4_t sum = {};
#pragma unroll
    for (int j = q * kEach; j < (q + 1) * kEach; ++j) sum = mfma_16x16x32<DT>(staged[0][16 * wave + f][(4 * j + part) ^ f], ones(), sum);
    if (f == 0) sums[0][q][4 * wave + part] = sum;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) read_x(0, e, x[e]);

  f32x4_t y[WT][MT] = {}, acc[2][MT] = {};
  float of_last = 0.f;        // the scale of the unit whose sums are still in acc
  u32x4_t w = sixteen_and<DT>(now.words[0][0], codes.mask, codes.bits);
  int buffer = 0;
  for (int b = 0; b < blocks; ++b) {
    const int after = buffer == 2 ? 0 : buffer + 1, b_next = b + 1 < blocks ? b + 1 : b;
    __syncthreads();          // the rows of blocks b and b + 1 and the sums of b are there, and what is of block b - 1 no longer read
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[0][m] = sums[b & 1][0][4 * m + part];
    // behind the last block too, which nobody reads: where all paths have the same loads, a wait is for the oldest alone
    stage(after == 2 ? 0 : after + 1, b + 2);
    fetch_rows(b + 3);
    uint32_t scale[WT][kGroups], off[WT][kGroups];
#pragma unroll
    for (int t = 0; t < WT; ++t) scales(t, scale[t], off[t]);
    fetch_scales(b_next);
    f32x4_t sum = {};
#pragma unroll
    for (int q = 0; q < kGroups; ++q)
#pragma unroll
      for (int t = 0; t < WT; ++t) {
        constexpr int kLast = WT - 1;
        const int unit = q * WT + t, t_last = (t + kLast) % WT;
        f32x4_t(&to)[MT] = acc[unit & 1], (&from)[MT] = acc[~unit & 1];
        u32x4_t x_sum;
        if (q == 0) x_sum = staged[after][16 * wave + f][(4 * t + part) ^ f];
        if constexpr (ZEROS) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[m][i] *= __uint_as_float(off[t][q]);
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int j = q * kEach + e;
          const uint32_t word = e + 1 < kEach ? now.words[t][j + 1] : t < kLast ? now.words[t + 1 < WT ? t + 1 : 0][q * kEach]
                                : q + 1 < kGroups ? now.words[0][(j + 1) % 4] : now.words[0][0];
          u32x4_t w_next;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            to[m] = mfma_16x16x32<DT>(x[e][m], w, to[m]);
            w_next[m] = sixteen_and_pair<DT>(word, m, codes.mask, codes.bits);
            // the last unit's sums in the first half, the next one's start in the second
            constexpr int kHalf = kEach * MT / 2;
            const int step = e * MT + m;
#pragma unroll
            for (int r = 0; r < kFlush; ++r) {
              const int at = step * kFlush + r, of = at / 4 % MT;
              if (at < 4 * MT) y[t_last][of][at % 4] = fmaf(of_last, from[of][at % 4], y[t_last][of][at % 4]);
              if (at < 4 * MT && at % 4 == 3) asm volatile("" : "+v"(y[t_last][of]));
            }
            if (unit + 1 < kGroups * WT && step >= kHalf && (kEach < 4 || step % 2 == 0)) {
#pragma unroll
              for (int r = 0; r < (kEach == 1 ? 2 : 1); ++r) {
                const int of = (step - kHalf) * 2 / kEach + r;
                from[of % MT] = sums[b & 1][(unit + 1) / WT % kGroups][4 * (of % MT) + part];
              }
            }
            // each matrix instruction with what goes on next to it, in this order
            asm volatile("" : "+v"(to[m]), "+v"(w_next[m]));
            __builtin_amdgcn_sched_barrier(0);
          }
          w = w_next;
          if (t == kLast) read_x(q + 1 < kGroups ? buffer : after, (q + 1) % kGroups * kEach + e, x[e]);
        }
        of_last = __uint_as_float(scale[t][q]);
        if (q + 1 == kGroups) fetch_words(t, b_next);
        if (q == 0) {
          sum = mfma_16x16x32<DT>(x_sum, ones(), t % kEach == 0 ? f32x4_t{} : sum);
          if ((t + 1) % kEach == 0 && f == 0) sums[(b + 1) & 1][t / kEach][4 * wave + part] = sum;
        }
      }
    buffer = after;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[WT - 1][m][i] = fmaf(of_last, acc[1][m][i], y[WT - 1][m][i]);
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

template <int DT, bool TWO, int GROUP>
void launch(const Rows4bit& g, int64_t slots, hipStream_t s) {
  for_slots(g, slots, [=](const Rows4bit& of, unsigned tiles) {
    const dim3 grid((unsigned)pieces_of(g.n, 16 * kFeatureWaves * (TWO ? kTiles / 2 : kTiles)), tiles);
    if (g.b[0].zeros) long_4bit_kernel<DT, TWO, GROUP, true><<<grid, kFeatureWaves * kWave, 0, s>>>(of);
    else long_4bit_kernel<DT, TWO, GROUP, false><<<grid, kFeatureWaves * kWave, 0, s>>>(of);
  });
}

template <int DT, bool TWO>
void by_group(const Rows4bit& g, int group, int64_t slots, hipStream_t s) {
  if (group == 32) launch<DT, TWO, 32>(g, slots, s);
  else if (group == 64) launch<DT, TWO, 64>(g, slots, s);
  else launch<DT, TWO, 128>(g, slots, s);
}

}  // namespace

int launch_long_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, hipStream_t s) {
  const bool two = g.b[1].words != nullptr;
  if (dtype == MBX_BF16) two ? by_group<MBX_BF16, true>(g, group, slots, s) : by_group<MBX_BF16, false>(g, group, slots, s);
  else two ? by_group<MBX_F16, true>(g, group, slots, s) : by_group<MBX_F16, false>(g, group, slots, s);
  return launch_status();
}

}  // namespace mbx
