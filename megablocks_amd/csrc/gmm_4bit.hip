// Weights in 4 bits with a scale (and a zero point) for every group of 32, 64 or 128 along the reduction: from 16- or 32-bit weights and back,
// and the experts' products with them.
//
// W [E, n, k] is kept in tiles of 16 features x 128 columns, in the order a wave multiplies them: 1 KiB in a row, 16 bytes a lane.  Lane
// 16 g + f has feature f; its word j has the columns 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7) of the tile, four bits each from the lowest, so that word
// j of all lanes is the operand of one v_mfma_f32_16x16x32 and a shift and a mask of a word give two neighbours in the halves of a register.
// scales [E, n / 16, k / group, 16] (zeros alike, a byte each): a code q stands for scale (q - zero), zero 8 without zeros.  n and k are rounded up to
// whole tiles; what lies past them is never used.
#include "common.h"

namespace mbx {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTileFeatures = 16, kTileColumns = 128, kTileWords = 256;

__device__ __host__ __forceinline__ int64_t tiles_of(int64_t n, int of) { return (n + of - 1) / of; }

struct Packed {
  const uint32_t* words;
  const void* scales;
  const uint8_t* zeros;
};

// ---- into 4 bits and back ----

constexpr int kPackThreads = 256;
constexpr int kPackFeatures = 64;          // of a workgroup: a tile for each wave

// rint(w / s), the quotient's exact value: ties to even.  inverse: 1 / (s lift)
template <int DT>
__device__ __forceinline__ float rounded_quotient(float w, float s, float inverse, float lift) {
  const float t = w * lift * inverse, q = rintf(t);
  if constexpr (DT == MBX_F32) {
    // t is off by up to 2^-20; where that may decide, in 64 bits
    if (fabsf(fabsf(t - q) - 0.5f) < 0x1p-16f) return (float)rint((double)w / (double)s);
    return q;
  } else {
    // of numbers of up to 11 bits a quotient is half way between two whole numbers or further than t is off by from there; w - s q is exact
    return fabsf(fmaf(-s, q, w)) == 0.5f * s ? 2.f * rintf(0.5f * t) : q;
  }
}

template <int DT> __device__ __forceinline__ float as_type(float v) { return Elem<DT>::to_f32(Elem<DT>::from_f32(v)); }

// The 32 weights of a lane (its tile's columns 32 j + 8 g + i) as codes and scales.  GROUP: columns.
template <int DT, int GROUP>
__device__ __forceinline__ void encode(const float (&w)[4][8], bool zero_points, u32x4_t& words, float (&scale)[128 / GROUP], int (&zero)[128 / GROUP]) {
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32;
#pragma unroll
  for (int p = 0; p < kGroups; ++p) {
    float low = 0.f, high = 0.f, bad = 0.f;
#pragma unroll
    for (int j = p * kEach; j < (p + 1) * kEach; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        low = fminf(low, w[j][i]);
        high = fmaxf(high, w[j][i]);
        bad = fmaf(w[j][i], 0.f, bad);   // NaN if one is not finite
      }
    // over the four lanes of a feature
#pragma unroll
    for (int step = 16; step <= 32; step += 16) {
      low = fminf(low, __shfl_xor(low, step));
      high = fmaxf(high, __shfl_xor(high, step));
      bad += __shfl_xor(bad, step);
    }
    float s = as_type<DT>(zero_points ? (high - low) / 15.f : fmaxf(high, -low) / 7.f);
    if (bad != 0.f || !(s < INFINITY)) s = NAN;
    const bool usable = s > 0.f;
    const float step = usable ? s : 1.f, lift = step < 0x1p-100f ? 0x1p64f : 1.f, inverse = 1.f / (step * lift);   // 1 / step may be infinite
    float z = 8.f;
    if (zero_points) {
      const float q = rounded_quotient<DT>(-low, step, inverse, lift);
      z = usable ? fminf(fmaxf(q, 0.f), 15.f) : 0.f;
    }
    scale[p] = s;
    zero[p] = (int)z;
#pragma unroll
    for (int j = p * kEach; j < (p + 1) * kEach; ++j) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf(rounded_quotient<DT>(w[j][i], step, inverse, lift) + z, 0.f), 15.f);
        word |= (usable ? (uint32_t)q : (uint32_t)z) << (4 * (i / 2 + 4 * (i & 1)));
      }
      words[j] = word;
    }
  }
}

// Where a workgroup of the two kernels is: 64 features, 128 columns of an expert
struct PackPlace {
  int64_t expert;
  int tile, block;   // of features (the wave's), of columns
};
__device__ __forceinline__ PackPlace pack_place(int64_t at, int feature_groups, int blocks) {
  PackPlace p;
  p.block = (int)(at % blocks);
  const int64_t rest = at / blocks;
  p.tile = (int)(rest % feature_groups) * (kPackFeatures / kTileFeatures) + (int)(threadIdx.x / kWave);
  p.expert = rest / feature_groups;
  return p;
}

constexpr int kPitch = kPackFeatures + 2;

// Weights [E, n, k] (TRANSPOSED: [E, k, n]) into words, scales and zeros.  What bounds it: one reading of the weights.  A lane's eight columns of a word
// are 16 bytes in a row of [n, k]; from [k, n] a workgroup's 64 features go through the LDS, whose pitch puts the four column groups of a read 8 (16) banks apart.
template <int DT, int GROUP, bool TRANSPOSED>
__global__ void __launch_bounds__(kPackThreads)
quantize_kernel(const void* __restrict__ weights, int64_t places, int n, int k, int feature_groups, int blocks, bool whole, uint32_t* __restrict__ words,
                void* __restrict__ scales, uint8_t* __restrict__ zeros) {
  typedef typename Elem<DT>::type E;
  __shared__ alignas(16) E staged[TRANSPOSED ? kTileColumns * kPitch : 1];
  const int lane = lane_id(), f = lane % 16, g = lane / 16, tiles = (n + 15) / 16;
  for (int64_t at = blockIdx.x; at < places; at += gridDim.x) {
    const PackPlace p = pack_place(at, feature_groups, blocks);
    const E* const matrix = (const E*)weights + p.expert * n * k;
    const int feature = p.tile * 16 + f, column = p.block * kTileColumns;
    float w[4][8];
    if constexpr (TRANSPOSED) {
      const int first = p.tile / 4 * kPackFeatures;
      __syncthreads();
      if (whole && first + kPackFeatures <= n) {
        constexpr int kEach = 16 / sizeof(E);
        for (int i = threadIdx.x; i < kTileColumns * kPackFeatures / kEach; i += kPackThreads) {
          const int row = i / (kPackFeatures / kEach), c = i % (kPackFeatures / kEach) * kEach;
          u32x4_t v = {0, 0, 0, 0};
          if (column + row < k) v = *(const u32x4_t*)(matrix + (int64_t)(column + row) * n + first + c);
          uint32_t* const to = (uint32_t*)(staged + row * kPitch + c);
#pragma unroll
          for (int q = 0; q < 4; ++q) to[q] = v[q];
        }
      } else {
        for (int i = threadIdx.x; i < kTileColumns * kPackFeatures; i += kPackThreads) {
          const int row = i / kPackFeatures, c = i % kPackFeatures;
          staged[row * kPitch + c] = column + row < k && first + c < n ? matrix[(int64_t)(column + row) * n + first + c] : E{};
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[j][i] = Elem<DT>::to_f32(staged[(32 * j + 8 * g + i) * kPitch + (p.tile % 4) * 16 + f]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = column + 32 * j + 8 * g;
        struct alignas(16) Piece { E v[8]; };
        if (whole) {
          Piece piece = {};
          if (feature < n && c < k) piece = *(const Piece*)(matrix + (int64_t)feature * k + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) w[j][i] = Elem<DT>::to_f32(piece.v[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[j][i] = feature < n && c + i < k ? Elem<DT>::to_f32(matrix[(int64_t)feature * k + c + i]) : 0.f;
        }
      }
    }
    u32x4_t code;
    float scale[128 / GROUP];
    int zero[128 / GROUP];
    encode<DT, GROUP>(w, zeros != nullptr, code, scale, zero);
    if (p.tile >= tiles) continue;   // no barrier behind this that the others wait at: the next place's are at its head, which all reach
    const int64_t tile = (p.expert * tiles + p.tile) * blocks + p.block;
    *(u32x4_t*)(words + tile * kTileWords + lane * 4) = code;
    if (g == 0) {
#pragma unroll
      for (int q = 0; q < 128 / GROUP; ++q) {
        ((E*)scales)[(tile * (128 / GROUP) + q) * 16 + f] = Elem<DT>::from_f32(scale[q]);
        if (zeros) zeros[(tile * (128 / GROUP) + q) * 16 + f] = (uint8_t)zero[q];
      }
    }
  }
}

// The values: the reverse
template <int DT, int GROUP, bool TRANSPOSED>
__global__ void __launch_bounds__(kPackThreads)
dequantize_kernel(const Packed from, int scale_dtype, int64_t places, int n, int k, int feature_groups, int blocks, bool whole, void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP;
  __shared__ alignas(16) E staged[TRANSPOSED ? kTileColumns * kPitch : 1];
  const int lane = lane_id(), f = lane % 16, g = lane / 16, tiles = (n + 15) / 16;
  for (int64_t at = blockIdx.x; at < places; at += gridDim.x) {
    const PackPlace p = pack_place(at, feature_groups, blocks);
    E* const matrix = (E*)out + p.expert * n * k;
    const int feature = p.tile * 16 + f, column = p.block * kTileColumns;
    E v[4][8] = {};
    if (p.tile < tiles) {
      const int64_t tile = (p.expert * tiles + p.tile) * blocks + p.block;
      const u32x4_t code = *(const u32x4_t*)(from.words + tile * kTileWords + lane * 4);
      float scale[kGroups], zero[kGroups];
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        const int64_t i = (tile * kGroups + q) * 16 + f;
        scale[q] = load_as_f32(from.scales, i, scale_dtype);
        zero[q] = from.zeros ? (float)from.zeros[i] : 8.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[j][i] = Elem<DT>::from_f32(((float)((code[j] >> (4 * (i / 2 + 4 * (i & 1)))) & 15u) - zero[j * kGroups / 4]) * scale[j * kGroups / 4]);
    }
    if constexpr (TRANSPOSED) {
      const int first = p.tile / 4 * kPackFeatures;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) staged[(32 * j + 8 * g + i) * kPitch + (p.tile % 4) * 16 + f] = v[j][i];
      __syncthreads();
      if (whole && first + kPackFeatures <= n) {
        constexpr int kEach = 16 / sizeof(E);
        for (int i = threadIdx.x; i < kTileColumns * kPackFeatures / kEach; i += kPackThreads) {
          const int row = i / (kPackFeatures / kEach), c = i % (kPackFeatures / kEach) * kEach;
          const uint32_t* const at = (const uint32_t*)(staged + row * kPitch + c);
          if (column + row < k) *(u32x4_t*)(matrix + (int64_t)(column + row) * n + first + c) = u32x4_t{at[0], at[1], at[2], at[3]};
        }
      } else {
        for (int i = threadIdx.x; i < kTileColumns * kPackFeatures; i += kPackThreads) {
          const int row = i / kPackFeatures, c = i % kPackFeatures;
          if (column + row < k && first + c < n) matrix[(int64_t)(column + row) * n + first + c] = staged[row * kPitch + c];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = column + 32 * j + 8 * g;
        struct alignas(16) Piece { E v[8]; };
        if (whole) {
          Piece piece;
#pragma unroll
          for (int i = 0; i < 8; ++i) piece.v[i] = v[j][i];
          if (feature < n && c < k) *(Piece*)(matrix + (int64_t)feature * k + c) = piece;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (feature < n && c + i < k) matrix[(int64_t)feature * k + c + i] = v[j][i];
        }
      }
    }
  }
}

// ---- products of few rows ----
//
// A wave has WT tiles of features (with a second matrix WT / 2 of each) and MT sixteens of rows, the waves of a workgroup a share of the columns each, a
// tile of 128 in turn; the shares are added up in the LDS, in order.  A word's codes become 16 + q in the activations' type by a shift, a mask and an or
// for two of them (bf16: the mantissa's upper four bits are its bits 3 - 6, fp16: 6 - 9); the products with a column of ones are the sums of the rows' group,
//   sum x scale (q - zero) = scale (sum x (16 + q) - (16 + zero) sum x)
// in fp32, where 16 + q costs four bits of 24 of which 16-bit activations have eleven.
constexpr int kRowsWaves = 4;

template <int DT>
__device__ __forceinline__ f32x4_t mfma_16x16x32(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
  typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
  if constexpr (DT == MBX_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// eight codes as 16 + q
template <int DT>
__device__ __forceinline__ u32x4_t sixteen_and(uint32_t word) {
  if constexpr (DT == MBX_BF16)
    return u32x4_t{(word << 3 & 0x00780078u) | 0x41804180u, (word >> 1 & 0x00780078u) | 0x41804180u, (word >> 5 & 0x00780078u) | 0x41804180u,
                   (word >> 9 & 0x00780078u) | 0x41804180u};
  else
    return u32x4_t{(word << 6 & 0x03c003c0u) | 0x4c004c00u, (word << 2 & 0x03c003c0u) | 0x4c004c00u, (word >> 2 & 0x03c003c0u) | 0x4c004c00u,
                   (word >> 6 & 0x03c003c0u) | 0x4c004c00u};
}

__device__ __forceinline__ float activated(float x, int act) {
  // x sigmoid(y): y = x (SiLU), or 2 sqrt(2 / pi) (x + 0.044715 x^3) (tanh-GELU)
  const float y = act == MBX_ACT_SILU ? x : 1.5957691216057308f * (x + 0.044715f * x * x * x);
  return x / (1.f + __expf(-y));
}

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
};

// Tile `slot` of up to `height` rows: its expert, first and end row, false past the last.  bins need not be trusted: bounds stay in [0, rows].
__device__ __forceinline__ bool find_rows(const Rows4bit& g, int slot, int height, int& expert, int64_t& first, int64_t& end) {
  const int lane = lane_id(), per = (g.num_groups + kWave - 1) / kWave;
  const auto bound = [&](int e) {   // rows before expert e
    const int64_t b = e <= 0 ? 0 : g.bins[e - 1];
    return b < 0 ? (int64_t)0 : b > g.rows ? g.rows : b;
  };
  const auto tiles = [&](int e) {
    const int64_t count = bound(e + 1) - bound(e);
    return count > 0 ? (int)((count + height - 1) / height) : 0;
  };
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (e < g.num_groups) mine += tiles(e);
  }
  const int upto = wave_inclusive_scan(mine);
  const uint64_t past = __ballot(upto > slot);
  if (past == 0) return false;
  const int at = __builtin_ctzll(past);
  int left = slot - lane_value(upto - mine, at);
  expert = at * per;
  for (;;) {
    const int count = __builtin_amdgcn_readfirstlane(tiles(expert));
    if (left < count || expert + 1 >= g.num_groups) break;
    left -= count;
    ++expert;
  }
  const int64_t begin = bound(expert), last = bound(expert + 1);
  first = begin + (int64_t)left * height;
  end = first + height < last ? first + height : last;
  return first < end;
}

template <int DT, int MT, int WT, bool TWO, int GROUP>
__global__ void __launch_bounds__(kRowsWaves * kWave)
rows_4bit_kernel(const Rows4bit g) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32;
  constexpr int kAhead = MT == 1 ? 4 : MT == 2 ? 2 : 1;    // tiles of columns whose loads are issued together
  constexpr int kFeatureTiles = TWO ? WT / 2 : WT;
  __shared__ float sums[kRowsWaves][WT * MT * 4][kWave];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), f = lane % 16, part = lane / 16;
  int expert;
  int64_t first, end;
  if (!find_rows(g, (int)blockIdx.y, 16 * MT, expert, first, end)) return;
  const int tiles = (g.n + 15) / 16, blocks = (g.k + 127) / 128, tile0 = (int)blockIdx.x * kFeatureTiles;
  // rows past the last are the last again: their results are not stored
  const uint16_t* row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    int64_t r = first + 16 * m + f;
    r = r < end ? r : end - 1;
    if (g.indices) {
      r = g.indices[r] / g.top_k;
      r = r < 0 ? 0 : r < g.a_rows ? r : g.a_rows - 1;
    }
    row[m] = (const uint16_t*)g.a + r * g.k;
  }
  f32x4_t y[WT][MT];
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const uint32_t one = DT == MBX_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const u32x4_t ones = {one, one, one, one};
  int64_t at[WT];      // the tile's first block
  Packed of[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    int tile = tile0 + (TWO ? t / 2 : t);
    tile = tile < tiles ? tile : tiles - 1;
    at[t] = ((int64_t)expert * tiles + tile) * blocks;
    of[t] = g.b[TWO ? t % 2 : 0];
  }
  for (int block = wave; block < blocks; block += kRowsWaves * kAhead) {
    u32x4_t words[kAhead][WT], x[kAhead][MT][4];
    uint32_t scale[kAhead][WT][kGroups], zero[kAhead][WT][kGroups];   // as they are in memory: nothing waits for a load in this loop
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int b = block + u * kRowsWaves;
      if (b >= blocks) continue;
#pragma unroll
      for (int t = 0; t < WT; ++t) words[u][t] = *(const u32x4_t*)(of[t].words + (at[t] + b) * kTileWords + lane * 4);
      const auto each_scale = [&](auto&& set) {
#pragma unroll
        for (int t = 0; t < WT; ++t)
#pragma unroll
          for (int q = 0; q < kGroups; ++q) set(t, q, ((at[t] + b) * kGroups + q) * 16 + f);
      };
      if (g.wide_scales) each_scale([&](int t, int q, int64_t i) { scale[u][t][q] = ((const uint32_t*)of[t].scales)[i]; });
      else each_scale([&](int t, int q, int64_t i) { scale[u][t][q] = ((const uint16_t*)of[t].scales)[i]; });
      if (of[0].zeros) each_scale([&](int t, int q, int64_t i) { zero[u][t][q] = of[t].zeros[i]; });
      else each_scale([&](int t, int q, int64_t) { zero[u][t][q] = 8; });
      const int c0 = b * kTileColumns + 8 * part;
      if ((b + 1) * kTileColumns <= g.k) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) __builtin_memcpy(&x[u][m][j], row[m] + c0 + 32 * j, 16);
      } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = c0 + 32 * j;
            if (c + 8 <= g.k) __builtin_memcpy(&x[u][m][j], row[m] + c, 16);
            else
#pragma unroll
              for (int i = 0; i < 4; ++i)
                x[u][m][j][i] = (c + 2 * i < g.k ? (uint32_t)row[m][c + 2 * i] : 0u) | (c + 2 * i + 1 < g.k ? (uint32_t)row[m][c + 2 * i + 1] << 16 : 0u);
          }
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (block + u * kRowsWaves >= blocks) continue;
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        f32x4_t of_ones[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          of_ones[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = q * kEach; j < (q + 1) * kEach; ++j) of_ones[m] = mfma_16x16x32<DT>(x[u][m][j], ones, of_ones[m]);
        }
#pragma unroll
        for (int t = 0; t < WT; ++t) {
          f32x4_t acc[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = q * kEach; j < (q + 1) * kEach; ++j) {
            const u32x4_t w = sixteen_and<DT>(words[u][t][j]);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = mfma_16x16x32<DT>(x[u][m][j], w, acc[m]);
          }
          const float s = g.wide_scales ? __uint_as_float(scale[u][t][q]) : Elem<DT>::to_f32(__builtin_bit_cast(E, (uint16_t)scale[u][t][q]));
          const float off = -16.f - (float)zero[u][t][q];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[t][m][i] = fmaf(s, fmaf(off, of_ones[m][i], acc[m][i]), y[t][m][i]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][(t * MT + m) * 4 + i][lane] = y[t][m][i];
  __syncthreads();
  // lane l, place i of a tile: row 4 (l / 16) + i, feature l % 16
  for (int v = wave; v < kFeatureTiles * MT * 4; v += kRowsWaves) {
    const int t = v / (MT * 4), rest = v % (MT * 4), m = rest / 4, i = rest % 4;
    const auto sum = [&](int tile) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWaves; ++w) s += sums[w][tile * MT * 4 + rest][lane];
      return s;
    };
    const int64_t r = first + 16 * m + 4 * part + i;
    const int feature = (tile0 + t) * 16 + f;
    if (r >= end || feature >= g.n) continue;
    float c = sum(TWO ? 2 * t : t);
    if (g.act >= 0) c = activated(c, g.act);
    if constexpr (TWO) c *= sum(2 * t + 1);
    ((E*)g.c)[r * g.n + feature] = Elem<DT>::from_f32(c);
  }
}

static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }

static bool is_dtype(int d) { return d == MBX_BF16 || d == MBX_F16 || d == MBX_F32; }

struct PackGrid {
  int feature_groups, blocks;
  int64_t places;
  unsigned grid;
  PackGrid(int64_t experts, int64_t n, int64_t k) {
    feature_groups = (int)tiles_of(n, kPackFeatures);
    blocks = (int)tiles_of(k, kTileColumns);
    places = experts * feature_groups * blocks;
    grid = (unsigned)(places < 256 * 64 ? places : 256 * 64);
  }
};

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

int mbx_quantize_4bit(const void* weights, int dtype, int num_experts, int n, int k, int layout, int group, void* words, void* scales, uint8_t* zeros,
                      mbx_stream_t stream) {
  if (!is_dtype(dtype) || num_experts < 0 || n < 0 || k < 0 || (layout != MBX_NT && layout != MBX_NN) || !group_ok(group)) return MBX_EINVAL;
  if (n > 0x7fffffff - 64 || k > 0x7fffffff - 128) return MBX_ERANGE;
  if (num_experts == 0 || n == 0 || k == 0) return 0;
  if (!weights || !words || !scales || ((uintptr_t)words & 15)) return MBX_EINVAL;
  const PackGrid p(num_experts, n, k);
  hipStream_t s = as_stream(stream);
  const int size = dtype_bytes(dtype), row = layout == MBX_NT ? k : n;
  const bool whole = ((uintptr_t)weights & 15) == 0 && row % (layout == MBX_NT ? 8 : 16 / size) == 0;
#define MBX_PACK_GROUP(KERNEL, DT, T, ...)                                                      \
  do {                                                                                          \
    if (group == 32) KERNEL<DT, 32, T><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__);            \
    else if (group == 64) KERNEL<DT, 64, T><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__);       \
    else KERNEL<DT, 128, T><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__);                       \
  } while (0)
#define MBX_PACK(KERNEL, ...)                                                                                                                \
  do {                                                                                                                                       \
    if (dtype == MBX_BF16) { if (layout == MBX_NN) MBX_PACK_GROUP(KERNEL, MBX_BF16, true, __VA_ARGS__); else MBX_PACK_GROUP(KERNEL, MBX_BF16, false, __VA_ARGS__); } \
    else if (dtype == MBX_F16) { if (layout == MBX_NN) MBX_PACK_GROUP(KERNEL, MBX_F16, true, __VA_ARGS__); else MBX_PACK_GROUP(KERNEL, MBX_F16, false, __VA_ARGS__); } \
    else { if (layout == MBX_NN) MBX_PACK_GROUP(KERNEL, MBX_F32, true, __VA_ARGS__); else MBX_PACK_GROUP(KERNEL, MBX_F32, false, __VA_ARGS__); } \
  } while (0)
  MBX_PACK(quantize_kernel, weights, p.places, n, k, p.feature_groups, p.blocks, whole, (uint32_t*)words, scales, zeros);
  return launch_status();
}

int mbx_dequantize_4bit(const void* words, const void* scales, const uint8_t* zeros, int scale_dtype, int num_experts, int n, int k, int layout, int group,
                        void* out, int dtype, mbx_stream_t stream) {
  if (!is_dtype(dtype) || !is_dtype(scale_dtype) || num_experts < 0 || n < 0 || k < 0 || (layout != MBX_NT && layout != MBX_NN) || !group_ok(group)) return MBX_EINVAL;
  if (n > 0x7fffffff - 64 || k > 0x7fffffff - 128) return MBX_ERANGE;
  if (num_experts == 0 || n == 0 || k == 0) return 0;
  if (!out || !words || !scales || ((uintptr_t)words & 15)) return MBX_EINVAL;
  const PackGrid p(num_experts, n, k);
  hipStream_t s = as_stream(stream);
  const int size = dtype_bytes(dtype), row = layout == MBX_NT ? k : n;
  const bool whole = ((uintptr_t)out & 15) == 0 && row % (layout == MBX_NT ? 8 : 16 / size) == 0;
  const Packed from = {(const uint32_t*)words, scales, zeros};
  MBX_PACK(dequantize_kernel, from, scale_dtype, p.places, n, k, p.feature_groups, p.blocks, whole, out);
#undef MBX_PACK
#undef MBX_PACK_GROUP
  return launch_status();
}

int mbx_gmm_4bit(const void* a, int64_t a_rows, const int32_t* indices, int top_k, const void* words, const void* scales, const uint8_t* zeros,
                 const void* words2, const void* scales2, const uint8_t* zeros2, int scale_dtype, int group, void* c, int dtype, const int32_t* bins,
                 int num_groups, int64_t rows, int k, int n, int act, mbx_stream_t stream) {
  if (!is_dtype(dtype) || !is_dtype(scale_dtype) || !group_ok(group) || num_groups < 0 || rows < 0 || k < 0 || n < 0 || act < -1 || act > MBX_ACT_GELU_TANH) return MBX_EINVAL;
  if (indices && (top_k <= 0 || a_rows < 0)) return MBX_EINVAL;
  if (words2 && (act < 0 || !zeros != !zeros2)) return MBX_EINVAL;
  if (dtype == MBX_F32 || (scale_dtype != dtype && scale_dtype != MBX_F32) || k == 0) return MBX_EUNSUPPORTED;
  if (rows > 0x7fffffff || n > 0x7fffffff - 64 || k > 0x7fffffff - 128) return MBX_ERANGE;
  if (rows == 0 || n == 0 || num_groups == 0) return 0;
  if (!a || !words || !scales || !c || !bins || (words2 && !scales2) || (indices && a_rows == 0)) return MBX_EINVAL;
  if (((uintptr_t)words | (uintptr_t)words2) & 15) return MBX_EINVAL;
  hipStream_t s = as_stream(stream);
  const Rows4bit g = {a, indices, a_rows, top_k, {{(const uint32_t*)words, scales, zeros}, {(const uint32_t*)words2, scales2, zeros2}}, scale_dtype == MBX_F32,
                      c, bins, num_groups, rows, k, n, act};
  const int64_t experts = rows < num_groups ? rows : num_groups, mean = ceil_div(rows, experts);
  const int mt = mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
  const int64_t slots = experts + rows / (16 * mt);
  if (slots > 65535) return MBX_EUNSUPPORTED;
#define MBX_ROWS_GROUP(DT, MT, WT, TWO)                                                                                          \
  do {                                                                                                                           \
    const dim3 grid((unsigned)tiles_of(n, 16 * (TWO ? WT / 2 : WT)), (unsigned)slots);                                           \
    if (group == 32) rows_4bit_kernel<DT, MT, WT, TWO, 32><<<grid, kRowsWaves * kWave, 0, s>>>(g);                               \
    else if (group == 64) rows_4bit_kernel<DT, MT, WT, TWO, 64><<<grid, kRowsWaves * kWave, 0, s>>>(g);                          \
    else rows_4bit_kernel<DT, MT, WT, TWO, 128><<<grid, kRowsWaves * kWave, 0, s>>>(g);                                          \
  } while (0)
#define MBX_ROWS(DT)                                                                                                             \
  do {                                                                                                                           \
    if (words2) {                                                                                                                \
      if (mt == 1) MBX_ROWS_GROUP(DT, 1, 2, true); else if (mt == 2) MBX_ROWS_GROUP(DT, 2, 2, true); else MBX_ROWS_GROUP(DT, 4, 2, true); \
    } else {                                                                                                                     \
      if (mt == 1) MBX_ROWS_GROUP(DT, 1, 2, false); else if (mt == 2) MBX_ROWS_GROUP(DT, 2, 2, false); else MBX_ROWS_GROUP(DT, 4, 2, false); \
    }                                                                                                                            \
  } while (0)
  if (dtype == MBX_BF16) MBX_ROWS(MBX_BF16);
  else MBX_ROWS(MBX_F16);
#undef MBX_ROWS
#undef MBX_ROWS_GROUP
  return launch_status();
}

}  // extern "C"
