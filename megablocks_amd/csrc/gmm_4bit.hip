// Weights in 4 bits with a scale (and a zero point) for every group of 32, 64 or 128 along the reduction: from 16- or 32-bit weights and back,
// and the choice of the products' kernels (gmm_4bit_rows.hip, gmm_4bit_tile.hip).
//
// W [E, n, k] is kept in tiles of 16 features x 128 columns, in the order a wave multiplies them: 1 KiB in a row, 16 bytes a lane.  Lane
// 16 g + f has feature f; its word j has the columns 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7) of the tile, four bits each from the lowest, so that word
// j of all lanes is the operand of one v_mfma_f32_16x16x32 and a shift and a mask of a word give two neighbours in the halves of a register.
// scales [E, n / 16, k / group, 16] (zeros alike, a byte each): a code q stands for scale (q - zero), zero 8 without zeros.  n and k are rounded up to
// whole tiles; what lies past them is never used.
#include "gmm_4bit.h"


namespace mbx {
namespace {

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

static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }

static bool is_dtype(int d) { return d == MBX_BF16 || d == MBX_F16 || d == MBX_F32; }

struct PackGrid {
  int feature_groups, blocks;
  int64_t places;
  unsigned grid;
  PackGrid(int64_t experts, int64_t n, int64_t k) {
    feature_groups = (int)pieces_of(n, kPackFeatures);
    blocks = (int)pieces_of(k, kTileColumns);
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
  if (rows > 0x7fffffff || n > 0x7fffffff - 1024 || k > 0x7fffffff - 256) return MBX_ERANGE;
  if (rows == 0 || n == 0 || num_groups == 0) return 0;
  if (!a || !words || !scales || !c || !bins || (words2 && !scales2) || (indices && a_rows == 0)) return MBX_EINVAL;
  if (((uintptr_t)words | (uintptr_t)words2) & 15) return MBX_EINVAL;
  hipStream_t s = as_stream(stream);
  const Rows4bit g = {a, indices, a_rows, top_k, {{(const uint32_t*)words, scales, zeros}, {(const uint32_t*)words2, scales2, zeros2}}, scale_dtype == MBX_F32,
                      c, bins, num_groups, rows, k, n, act};
  // up to 12 rows an expert in the mean of those that can have some the one kernel, then the other (us, one / other: 8 gated experts of [4096, 14336], 8 rows
  // 93 / 115, 16 rows 143 / 119; 64 of [2048, 1408], 3 rows 40 / 46, 15 rows 62 / 48)
  const int64_t experts = rows < num_groups ? rows : num_groups;
  const bool few = rows <= 12 * experts;
  const int64_t slots = experts + rows / (few ? 16 : 32);
  if (slots > 65535) return MBX_EUNSUPPORTED;
  return few ? launch_rows_4bit(g, dtype, group, slots, experts, s) : launch_tiles_4bit(g, dtype, group, slots, s);
}

}  // extern "C"
