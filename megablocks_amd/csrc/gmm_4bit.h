// Products with 4-bit weights: what their kernels share.  How the weights are kept: gmm_4bit.hip.
#pragma once

#include "common.h"

namespace mbx {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTileFeatures = 16, kTileColumns = 128, kTileWords = 256;

struct Packed {
  const uint32_t* words;
  const void* scales;
  const uint8_t* zeros;
};

struct Rows4bit {
  const void* a;
  const int32_t* indices;   // NULL: row r of a is row r
  int64_t a_rows;
  int top_k;
  Packed b[2];
  int wide_scales;          // fp32 instead of the activations' type
  void* c;
  const int32_t* bins;
  int num_groups;
  int64_t rows;
  int k, n, act;            // act < 0: none
  int first_slot;           // the launch's first tile of rows
};

// The kernels: of tiles of 16 rows (few rows an expert), 32 (dozens) and 64 (hundreds), `slots` of them at most.  dtype, group, zeros and whether there is a
// second matrix are the arguments'.
int launch_rows_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, int64_t experts, hipStream_t s);
int launch_tiles_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, hipStream_t s);
int launch_long_4bit(const Rows4bit& g, int dtype, int group, int64_t slots, hipStream_t s);

namespace {

template <int DT>
__device__ __forceinline__ f32x4_t mfma_16x16x32(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
  typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
  if constexpr (DT == MBX_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Eight codes as 16 + q.  mask and bits: kNibbles and kSixteens of the type, in registers that the compiler does not know the contents of (as numbers in the
// instruction they keep the mask and the or from being one).
template <int DT> struct Codes;
template <> struct Codes<MBX_BF16> { static constexpr uint32_t kNibbles = 0x00780078u, kSixteens = 0x41804180u; static constexpr int kUp = 3; };
template <> struct Codes<MBX_F16> { static constexpr uint32_t kNibbles = 0x03c003c0u, kSixteens = 0x4c004c00u; static constexpr int kUp = 6; };
template <int DT>
__device__ __forceinline__ uint32_t sixteen_and_pair(uint32_t word, int i, uint32_t mask, uint32_t bits) {
  const int up = Codes<DT>::kUp - 4 * i;
  return ((up >= 0 ? word << (up >= 0 ? up : 0) : word >> (up < 0 ? -up : 0)) & mask) | bits;
}
template <int DT>
__device__ __forceinline__ u32x4_t sixteen_and(uint32_t word, uint32_t mask, uint32_t bits) {
  u32x4_t out;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = sixteen_and_pair<DT>(word, i, mask, bits);
  return out;
}

__device__ __forceinline__ float activated(float x, int act) {
  // x sigmoid(y): y = x (SiLU), or 2 sqrt(2 / pi) (x + 0.044715 x^3) (tanh-GELU)
  const float y = act == MBX_ACT_SILU ? x : 1.5957691216057308f * (x + 0.044715f * x * x * x);
  return x / (1.f + __expf(-y));
}

// The workgroup's tile of up to `height` rows: its expert, first and end row, false past the last.  bins need not be trusted: bounds stay in [0, rows], and a lane
// counts no further than it has the slot, so that falling bins of many experts, each with all rows, do not pass 32 bits: up to the lane that has it sums are exact.
__device__ __forceinline__ bool find_rows(const Rows4bit& g, int height, int& expert, int& first, int& end) {
  const int slot = g.first_slot + (int)blockIdx.y;
  const int lane = lane_id(), per = (g.num_groups + kWave - 1) / kWave, rows = (int)g.rows;
  const auto clipped = [&](int b) { return b < 0 ? 0 : b > rows ? rows : b; };
  const auto bound = [&](int e) { return e <= 0 ? 0 : clipped(g.bins[e - 1]); };   // rows before expert e
  const auto tiles = [&](int begin, int last) { return last > begin ? (last - begin + height - 1) / height : 0; };
  int mine = 0, begin = 0, last = 0;
  if (per == 1) {   // an expert a lane: what is found below is in its lane's registers
    const int at = lane < g.num_groups ? lane : g.num_groups - 1;
    last = clipped(g.bins[at]);
    begin = __builtin_amdgcn_update_dpp(0, last, 0x138, 0xf, 0xf, false);   // of the lane below, 0 in lane 0
    mine = lane < g.num_groups ? tiles(begin, last) : 0;
  } else {
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < g.num_groups && mine <= slot) mine += tiles(bound(e), bound(e + 1));
    }
  }
  const int upto = wave_inclusive_scan(mine);
  const uint64_t past = __ballot(upto > slot);
  if (past == 0) return false;
  const int at = __builtin_ctzll(past);
  int left = slot - lane_value(upto - mine, at);
  expert = at * per;
  if (per == 1) {
    begin = lane_value(begin, at);
    last = lane_value(last, at);
  } else {
    for (;;) {
      begin = __builtin_amdgcn_readfirstlane(bound(expert));
      last = __builtin_amdgcn_readfirstlane(bound(expert + 1));
      const int count = tiles(begin, last);
      if (left < count || expert + 1 >= g.num_groups) break;
      left -= count;
      ++expert;
    }
  }
  first = begin + left * height;
  end = last - first < height ? last : first + height;
  return first < end;
}

// An address in device memory that is the wave's, as the compiler does not see by itself: loads then add a lane's place to it as 32 bits.
typedef const __attribute__((address_space(1))) char* wave_ptr;
__device__ __forceinline__ wave_ptr of_wave(const void* p) {
  const uint64_t u = (uint64_t)p;
  return (wave_ptr)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u));
}
template <typename T>
__device__ __forceinline__ T load_at(wave_ptr base, int64_t of_wave_bytes, uint32_t of_lane) {
  return *(const __attribute__((address_space(1))) T*)(base + of_wave_bytes + of_lane);
}

// A value for every lane from the lane of the same f in row q of 16 lanes, for all four rows q: a block's scales are one load of 64 lanes.
template <int GROUPS>
__device__ __forceinline__ void spread(uint32_t v, uint32_t (&of)[GROUPS]) {
  if constexpr (GROUPS == 1) {
    of[0] = v;
  } else if constexpr (GROUPS == 2) {      // rows 0, 1, 0, 1
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    of[0] = p[0];
    of[1] = p[1];
  } else {                                 // rows 0, 1, 2, 3
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const auto low = __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false), high = __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false);
    of[0] = low[0];
    of[1] = low[1];
    of[2] = high[0];
    of[3] = high[1];
  }
}

inline int64_t pieces_of(int64_t n, int of) { return (n + of - 1) / of; }

// launch(g, rows of the grid) for all slots, 65535 at a time
template <typename F>
void for_slots(Rows4bit g, int64_t slots, F&& launch) {
  for (int64_t first = 0; first < slots; first += 65535) {
    g.first_slot = (int)first;
    launch(g, (unsigned)(slots - first < 65535 ? slots - first : 65535));
  }
}

// A wave's WT tiles of weights of one expert (TWO: every other one of the second matrix), a block of 128 columns at a time.
template <int DT, int WT, bool TWO, int GROUP>
struct Weights4bit {
  static constexpr int kGroups = 128 / GROUP;
  struct Block {
    u32x4_t words[WT];
    uint32_t scale[WT], zero[WT];   // as they are in memory: nothing waits for a load before the block is multiplied
  };
  wave_ptr words_at[WT], scales_at[WT], zeros_at[WT];
  uint32_t word_lane, scale_lane, scale_at, half_up, half_mask;
  int scale_shift, groups;
  bool wide, with_zeros;

  __device__ __forceinline__ Weights4bit(const Rows4bit& g, int expert, int tile0, int tiles, int blocks) {
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      int tile = tile0 + (TWO ? t / 2 : t);
      tile = tile < tiles ? tile : tiles - 1;     // past the last: the last again, not stored
      const Packed of = g.b[TWO ? t % 2 : 0];
      const int64_t at = ((int64_t)expert * tiles + tile) * blocks;
      words_at[t] = of_wave(of.words + at * kTileWords);
      scales_at[t] = of_wave((const char*)of.scales + at * kGroups * 16 * (g.wide_scales ? 4 : 2));
      zeros_at[t] = of_wave(of.zeros ? of.zeros + at * kGroups * 16 : nullptr);
    }
    word_lane = (uint32_t)lane_id() * 16;
    scale_lane = (uint32_t)lane_id() % (kGroups * 16);
    wide = g.wide_scales;
    with_zeros = zeros_at[0] != nullptr;
    // The piece of 4 bytes with the lane's scale, one load whatever the type (of two in branches the second waits for the first); as 16 bits the lane's half
    // is shifted up and the other cut off
    scale_shift = wide ? 2 : 1;
    scale_at = scale_lane << scale_shift & ~3u;
    half_up = wide || scale_lane % 2 ? 0 : 16;
    half_mask = wide ? ~0u : 0xffff0000u;
    groups = (g.k + GROUP - 1) / GROUP;
  }

  // ONCE: read by nobody else, kept out of the caches (60 MiB of weights read alone: 9.7 us, with plain loads 10.9; 480 MiB: 69, 78)
  template <bool ONCE>
  __device__ __forceinline__ void fetch_words(Block& to, int t, int b) const {
    const auto at = (const __attribute__((address_space(1))) u32x4_t*)(words_at[t] + (int64_t)b * (kTileWords * 4) + word_lane);
    if constexpr (ONCE) to.words[t] = __builtin_nontemporal_load(at);
    else to.words[t] = *at;
  }
  __device__ __forceinline__ void fetch_scales(Block& to, int b) const {
#pragma unroll
    for (int t = 0; t < WT; ++t) to.scale[t] = load_at<uint32_t>(scales_at[t], (int64_t)b * (kGroups * 16) << scale_shift, scale_at);
    if (with_zeros) {
#pragma unroll
      for (int t = 0; t < WT; ++t) to.zero[t] = load_at<uint8_t>(zeros_at[t], (int64_t)b * (kGroups * 16), scale_lane);
    }
  }
  template <bool ONCE>
  __device__ __forceinline__ void fetch(Block& to, int b) const {
#pragma unroll
    for (int t = 0; t < WT; ++t) fetch_words<ONCE>(to, t, b);
    fetch_scales(to, b);
  }

  // The bits of a scale's piece that are used in block b: none of groups that lie wholly past k, whose sums are 0, but 0 times a scale that is not finite is not
  __device__ __forceinline__ uint32_t mask_of(int b) const { return kGroups > 1 && scale_lane >= (uint32_t)(groups - b * kGroups) * 16 ? 0u : half_mask; }
  // scale and -(16 + zero) of the lane's feature for each group; mask: mask_of the block
  __device__ __forceinline__ void scales(const Block& of, int t, uint32_t mask, uint32_t (&scale)[kGroups], uint32_t (&off)[kGroups]) const {
    const uint32_t raw = (of.scale[t] << half_up) & mask;
    float s = __uint_as_float(raw);
    if constexpr (DT == MBX_F16) s = wide ? s : Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(raw >> 16)));
    spread<kGroups>(__float_as_uint(s), scale);
    spread<kGroups>(__float_as_uint(with_zeros ? -16.f - (float)of.zero[t] : -24.f), off);
  }
};

// mask and bits of sixteen_and
template <int DT>
struct CodeBits {
  uint32_t mask = Codes<DT>::kNibbles, bits = Codes<DT>::kSixteens;
  __device__ __forceinline__ CodeBits() {
    asm("" : "+s"(mask));
    asm("" : "+v"(bits));
  }
};
// Eight times v, which the type holds
template <int DT>
__device__ __forceinline__ u32x4_t all_of(float v) {
  const uint32_t one = __builtin_bit_cast(uint16_t, Elem<DT>::from_f32(v)), two = one << 16 | one;
  return u32x4_t{two, two, two, two};
}
template <int DT>
__device__ __forceinline__ u32x4_t ones_of() { return all_of<DT>(1.f); }

// Columns c ... c + 7 of a row of k, zeros past its end
__device__ __forceinline__ void read_columns(const uint16_t* row, int c, int k, u32x4_t& to) {
  if (c + 8 <= k) __builtin_memcpy(&to, row + c, 16);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      to[i] = (c + 2 * i < k ? (uint32_t)row[c + 2 * i] : 0u) | (c + 2 * i + 1 < k ? (uint32_t)row[c + 2 * i + 1] << 16 : 0u);
}
// Row r of the product's rows
__device__ __forceinline__ const uint16_t* row_of(const Rows4bit& g, int64_t r) {
  if (g.indices) {
    r = g.indices[r] / g.top_k;
    r = r < 0 ? 0 : r < g.a_rows ? r : g.a_rows - 1;
  }
  return (const uint16_t*)g.a + r * g.k;
}

}  // namespace
}  // namespace mbx
