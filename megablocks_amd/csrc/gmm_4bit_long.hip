// Products of hundreds to thousands of rows an expert with 4-bit weights.
//
// A workgroup has 64 rows, four waves with 64 features each (with a second matrix 32 of each), all columns; rows, weights and the start of the sums as in
// gmm_4bit_tile.hip.  A wave multiplies by 32 x 32 x 16: a step of 16 columns is four matrix instructions, and next to each, in this order, a quarter of the
// next step's operands is made of the codes; a group's sums are scaled and added up (64 instructions) while the next group's start is on its way.  A lane's
// words of half a block are loaded half a block ahead, rows three blocks.  That is the 256 registers there are for two waves on a SIMD; where the rows are
// is kept in the LDS for that.
//
// What bounds it: issuing, and waiting with two waves a SIMD.  A SIMD issues a vector instruction every 4 cycles, and next to them a matrix instruction of 32 x 32 x 16
// costs 2.4 such places, one of 16 x 16 x 32, half the work, 2 (measured); 36 of them and some 290 others a block are 370 places of 4 cycles, 2960 for both waves, where a
// block takes 4100 cycles of a clock that is down to 1.84 GHz.  Counted, 1024 rows an expert: the matrix pipe is busy in 52 % of the cycles, 63 % of the places are
// taken; of its time a wave issues vector instructions for 33 %, waits for its turn to issue for 38 %, and for loads, the LDS or the barrier for 17 %.  128 rows: 46 %, 56 %;
// 33, 36 and 20 %.
// First products of 8 gated experts of [4096, 14336], 128 / 256 / 512 / 1024 rows an expert: 345 / 608 / 1088 / 2030 us (698 / 792 / 885 / 948 TFLOP/s); by
// 16 x 16 x 32 351 / 623 / 1121 / 2107; 128 rows a workgroup with one wave a SIMD and all 512 registers 2245; values made in 16 bits, which rounds each weight,
// and multiplied by the grouped kernels 2016 for 1024 rows.  Workgroups of an XCD by 16 tiles of rows and a few features 2001, but 64 experts of [2048, 1408],
// whose features do not divide by the XCDs, 405 -> 493.  Groups of 32, 512 rows of 8 experts of [14336, 4096]: 784 us (614 TFLOP/s): four times the sums.
#include "gmm_4bit.h"

namespace mbx {
namespace {

constexpr int kFeatureWaves = 4, kRows = 64, kWaveFeatures = 64;   // a workgroup: 64 rows, four waves with 64 features (with a second matrix 32 of each)

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f32x16_t mfma_32x32x16(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
  typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
  typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
  if constexpr (DT == MBX_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

template <int DT, bool TWO, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kFeatureWaves * kWave, 2)
long_4bit_kernel(const Rows4bit g) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32, kSteps = GROUP / 16;
  __shared__ u32x4_t staged[3][kRows][16];
  __shared__ f32x4_t sums[2][kGroups][kRows / 4];
  __shared__ uint64_t rows_at[kRows];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n32 = lane % 32, h = lane / 32, f = lane % 16, part = lane / 16;   // of 32 x 32 x 16 products; of the sums' 16 x 16 x 32
  int expert, first, end;
  if (!find_rows(g, kRows, expert, first, end)) return;   // alike for all waves: none is left at a barrier
  const int tiles = (g.n + 15) / 16, blocks = (g.k + 127) / 128, tile0 = ((int)blockIdx.x * kFeatureWaves + wave) * (TWO ? 2 : 4);

  // The wave's two tiles of 32 features, two of the 16 in memory each; past the last the last again, not stored
  wave_ptr words_at[2], scales_at[2], zeros_at[2];
  uint32_t tile_of[2];          // the lane's second 16, in tiles
  const bool wide = g.wide_scales;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int tile = tile0 + (TWO ? 0 : 2 * t), base = tile < tiles ? tile : tiles - 1;
    tile_of[t] = n32 >= 16 && base + 1 < tiles ? 1 : 0;
    const Packed of = g.b[TWO ? t : 0];
    const int64_t at = ((int64_t)expert * tiles + base) * blocks;
    words_at[t] = of_wave(of.words + at * kTileWords);
    scales_at[t] = of_wave((const char*)of.scales + at * kGroups * 16 * (wide ? 4 : 2));
    zeros_at[t] = of_wave(ZEROS ? of.zeros + at * kGroups * 16 : nullptr);
  }
  // what the call has checked: two tiles' words are less than 2^32 bytes
  uint32_t word_at[2], scale_at[2], zero_at[2];
  const int scale_shift = wide ? 2 : 1;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    word_at[t] = tile_of[t] * (uint32_t)blocks * (kTileWords * 4) + (uint32_t)(16 * h + f) * 16;
    zero_at[t] = tile_of[t] * (uint32_t)blocks * (kGroups * 16) + (uint32_t)f;
    scale_at[t] = zero_at[t] << scale_shift & ~3u;      // the piece of 4 bytes with the scale
  }
  const uint32_t half_up = wide || f % 2 ? 0 : 16, half_mask = wide ? ~0u : 0xffff0000u;
  // words[t][p][i]: of steps 4 i + p and 4 i + 2 + p
  u32x2_t words[2][2][2];
  uint32_t scale_raw[2], zero_raw[2];     // of the next group
  const auto fetch_words = [&](int i, int b) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = 0; p < 2; ++p) words[t][p][i] = load_at<u32x2_t>(words_at[t], 0, word_at[t] + (uint32_t)b * (kTileWords * 4) + (uint32_t)(p * 512 + i * 8));
  };
  const auto word_of = [&](int t, int s) { return words[t][s % 2][s / 4][s / 2 % 2]; };
  const auto fetch_scales = [&](int group) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      scale_raw[t] = load_at<uint32_t>(scales_at[t], 0, scale_at[t] + ((uint32_t)group * 16 << scale_shift));
      if constexpr (ZEROS) zero_raw[t] = load_at<uint8_t>(zeros_at[t], 0, zero_at[t] + (uint32_t)group * 16);
    }
  };
  // of groups that lie wholly past k 0: their sums are 0, but 0 times a scale that is not finite is not
  const auto scale_of = [&](int t, int group) {
    const uint32_t raw = (scale_raw[t] << half_up) & (kGroups > 1 && group * GROUP >= g.k ? 0u : half_mask);
    if constexpr (DT == MBX_F16) return wide ? __uint_as_float(raw) : Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(raw >> 16)));
    else return __uint_as_float(raw);
  };

  // thread i stages piece i % 16 of rows i / 16, i / 16 + 16, ...; rows past the last are the last again
  constexpr int kStaged = kRows / 16;
  const int piece = (int)threadIdx.x % 16, stage_row = (int)threadIdx.x / 16;
  if (threadIdx.x < kRows) {      // where the rows are, in the LDS: registers are short
    const int r = first + (int)threadIdx.x;
    rows_at[threadIdx.x] = (uint64_t)row_of(g, r < end ? r : end - 1);
  }
  __syncthreads();
  struct __attribute__((packed, aligned(2))) Piece { u32x4_t v; };      // rows need not begin at whole pieces
  u32x4_t x_next[kStaged];
  const auto fetch_rows = [&](int b) {
    const int c = b * kTileColumns + 8 * piece;      // rows are whole pieces: past the last, the first
#pragma unroll
    for (int m = 0; m < kStaged; ++m)
      x_next[m] = ((const __attribute__((address_space(1))) Piece*)(rows_at[16 * m + stage_row] + (uint32_t)(c < g.k ? c : 0) * 2))->v;
  };
  const auto stage = [&](int buffer, int b) {
    if (b + 1 == blocks && b * kTileColumns + 8 * piece >= g.k) {
#pragma unroll
      for (int m = 0; m < kStaged; ++m) x_next[m] = u32x4_t{};
    }
#pragma unroll
    for (int m = 0; m < kStaged; ++m) staged[buffer][16 * m + stage_row][piece ^ stage_row] = x_next[m];
  };
  const auto ones = [] {      // made where they are used: registers are short
    uint32_t one = all_of<DT>(ZEROS ? 1.f : -24.f)[0];
    asm volatile("" : "+v"(one));
    return u32x4_t{one, one, one, one};
  };
  const CodeBits<DT> codes;
  const auto read_x = [&](int buffer, int s, u32x4_t (&to)[2]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) to[m] = staged[buffer][32 * m + n32][(2 * s + h) ^ f];
  };

  fetch_rows(0);
  stage(0, 0);
  fetch_rows(1);
  stage(1, 1);
  fetch_rows(2);
  fetch_scales(0);
  fetch_words(0, 0);
  fetch_words(1, 0);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kGroups; ++q) {
    f32x4_t sum = {};
#pragma unroll
    for (int j = q * kEach; j < (q + 1) * kEach; ++j) sum = mfma_16x16x32<DT>(staged[0][16 * wave + f][(4 * j + part) ^ f], ones(), sum);
    if (f == 0) sums[0][q][4 * wave + part] = sum;
  }
  u32x4_t x[2], w[2];
  read_x(0, 0, x);
#pragma unroll
  for (int t = 0; t < 2; ++t) w[t] = sixteen_and<DT>(word_of(t, 0), codes.mask, codes.bits);
  f32x16_t y[2][2] = {}, acc[2][2] = {};
  float of_last[2] = {0.f, 0.f};     // the scales of the group whose sums are still in acc
  const auto add_up = [&] {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[t][m][i] = fmaf(of_last[t], acc[t][m][i], y[t][m][i]);
        asm volatile("" : "+v"(y[t][m]));
      }
  };
  __builtin_amdgcn_s_waitcnt(0x0f70);     // all loads: the loop's waits are then for its own alone, in their order
  int buffer = 0;
  for (int b = 0; b < blocks; ++b) {
    const int after = buffer == 2 ? 0 : buffer + 1, b_next = b + 1 < blocks ? b + 1 : b;
    __syncthreads();          // the rows of blocks b and b + 1 and the sums of b are there, and what is of block b - 1 no longer read
    f32x4_t sum = {};
    u32x4_t x_sum;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      f32x16_t base[2];
      const auto read_base = [&](int m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4_t four = sums[b & 1][q][8 * m + 2 * i + h];
#pragma unroll
          for (int r = 0; r < 4; ++r) base[m][4 * i + r] = four[r];
        }
      };
      read_base(0);
      add_up();
      if (q == 0) {
        // behind the last block too, which nobody reads: where all paths have the same loads, a wait is for the oldest alone
        stage(after == 2 ? 0 : after + 1, b + 2);
        fetch_rows(b + 3);
      }
      float off[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        of_last[t] = scale_of(t, b * kGroups + q);
        if constexpr (ZEROS) off[t] = -16.f - (float)zero_raw[t];
      }
      fetch_scales(q + 1 < kGroups ? b * kGroups + q + 1 : b_next * kGroups);
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        const int s = q * kSteps + e;
        u32x4_t x_then[2], w_then[2];
        read_x(s == 7 ? after : buffer, (s + 1) % 8, x_then);
        if (s % 2 == 0) x_sum = staged[after][16 * wave + f][(2 * s + part) ^ f];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (e == 0) {
              f32x16_t start = base[m];
              if constexpr (ZEROS)
#pragma unroll
                for (int i = 0; i < 16; ++i) start[i] *= off[t];
              acc[t][m] = mfma_32x32x16<DT>(x[m], w[t], start);
            } else {
              acc[t][m] = mfma_32x32x16<DT>(x[m], w[t], acc[t][m]);
            }
            // the next step's operands: half of one next to each
#pragma unroll
            for (int i = 2 * t; i < 2 * t + 2; ++i) w_then[m][i] = sixteen_and_pair<DT>(word_of(m, (s + 1) % 8), i, codes.mask, codes.bits);
            asm volatile("" : "+v"(acc[t][m]), "+v"(w_then[m][2 * t]), "+v"(w_then[m][2 * t + 1]));
            __builtin_amdgcn_sched_barrier(0);
            if (e == 0 && m == 0 && t == 1) read_base(1);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] = x_then[i];
          w[i] = w_then[i];
        }
        if (s == 2) fetch_words(0, b_next);       // words of steps 0 - 3: the last operand has been made
        if (s == 6) fetch_words(1, b_next);
        if (s % 2 == 1) {
          sum = mfma_16x16x32<DT>(x_sum, ones(), s / 2 % kEach == 0 ? f32x4_t{} : sum);
          if ((s / 2 + 1) % kEach == 0 && f == 0) sums[(b + 1) & 1][s / 2 / kEach][4 * wave + part] = sum;
        }
      }
    }
    buffer = after;
  }
  add_up();
#pragma unroll
  for (int t = 0; t < (TWO ? 1 : 2); ++t)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = first + 32 * m + 8 * (i / 4) + 4 * h + i % 4, feature = (tile0 + 2 * t) * 16 + n32;
        float c = y[t][m][i];
        if (g.act >= 0) c = activated(c, g.act);
        if constexpr (TWO) c *= y[1][m][i];
        if (r < end && feature < g.n) ((E*)g.c)[(int64_t)r * g.n + feature] = Elem<DT>::from_f32(c);
      }
}

template <int DT, bool TWO, int GROUP>
void launch(const Rows4bit& g, int64_t slots, hipStream_t s) {
  for_slots(g, slots, [=](const Rows4bit& of, unsigned tiles) {
    const dim3 grid((unsigned)pieces_of(g.n, kFeatureWaves * kWaveFeatures / (TWO ? 2 : 1)), tiles);
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
