// Weights in 4 bits with a scale (and a zero point) for every group of 32, 64 or 128 along the reduction: from 16- or 32-bit weights and back,
// and the choice of the products' kernels (gmm_4bit_rows.hip, gmm_4bit_tile.hip, gmm_4bit_long.hip).
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

// rint(w / s) of the exact quotient, halves to even, plus a whole number: even if EVEN, which then costs nothing.  inverse: 1 / s.
template <int DT, bool EVEN>
__device__ __forceinline__ float rounded_quotient(float w, float s, float inverse, float add) {
  if constexpr (DT == MBX_F32) {
    const float t = w * inverse, q = rintf(t);
    // t is off by up to 2^-20; where that may decide, in 64 bits
    return (fabsf(fabsf(t - q) - 0.5f) < 0x1p-16f ? (float)rint((double)w / (double)s) : q) + add;
  } else {
    // of two numbers of up to 11 bits the quotient is half way between two whole numbers or 2^-13 and more from there: to whole multiples of 2^-14, the last
    // place of numbers from 512 to 1024, a quotient that is off by 2^-20 becomes the half that it is, or stays on its side
    constexpr float kSnap = 768.f;
    const float snapped = fmaf(w, inverse, kSnap);
    return EVEN ? rintf(snapped - (kSnap - add)) : rintf(snapped - kSnap) + add;
  }
}

template <int DT> __device__ __forceinline__ float as_type(float v) { return Elem<DT>::to_f32(Elem<DT>::from_f32(v)); }

// The 32 weights of a lane (its tile's columns 32 j + 8 g + i) as codes and scales.  GROUP: columns.
template <int DT, int GROUP, bool ZEROS>
__device__ __forceinline__ void encode(const float (&w)[4][8], u32x4_t& words, float (&scale)[128 / GROUP], int (&zero)[128 / GROUP]) {
  constexpr int kGroups = 128 / GROUP, kEach = GROUP / 32;
#pragma unroll
  for (int p = 0; p < kGroups; ++p) {
    float low = 0.f, high = 0.f;     // without zero points high is the largest size
    bool bad = false;                // one is not a number
#pragma unroll
    for (int j = p * kEach; j < (p + 1) * kEach; ++j)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float a = w[j][i], b = w[j][i + 1];
        if constexpr (ZEROS) {
          low = fminf(fminf(a, b), low);
          high = fmaxf(fmaxf(a, b), high);
        } else {
          high = fmaxf(fmaxf(fabsf(a), fabsf(b)), high);
        }
        bad |= __builtin_isunordered(a, b);
      }
    // over the four lanes of a feature
    const uint64_t lanes = __ballot(bad);
    bad = ((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) >> (lane_id() % 16)) & 1;
    const auto over = [](float v, auto&& op) {
      const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
      const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      return op(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    };
    high = over(high, [](float a, float b) { return fmaxf(a, b); });
    if constexpr (ZEROS) low = over(low, [](float a, float b) { return fminf(a, b); });
    float s = ZEROS ? (high - low) * (1.f / 15.f) : high * (1.f / 7.f);     // by the reciprocal in 32 bits, as torch divides by a number
    asm("" : "+v"(s));                            // rounded there: a product and a rounding to fp16 in one instruction are rounded once
    s = as_type<DT>(s);
    if (s < 0x1p-126f) s = 0.f;                   // no normal number of 32 bits: its inverse may be none
    if (bad || !(s < INFINITY)) s = NAN;
    const bool usable = s > 0.f;
    const float inverse = 1.f / (usable ? s : 1.f);
    float z = 8.f;
    if constexpr (ZEROS) z = usable ? fminf(fmaxf(rounded_quotient<DT, true>(-low, s, inverse, 0.f), 0.f), 15.f) : 0.f;
    scale[p] = s;
    zero[p] = (int)z;
    const uint32_t none = (uint32_t)(int)z * 0x11111111u;
#pragma unroll
    for (int j = p * kEach; j < (p + 1) * kEach; ++j) {
      float half[2];       // of the word, a number below 2^16
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 6; i >= 0; i -= 2) {
          const float q = __builtin_amdgcn_fmed3f(rounded_quotient<DT, !ZEROS>(w[j][i + h], s, inverse, z), 0.f, 15.f);
          half[h] = i == 6 ? q : fmaf(half[h], 16.f, q);
        }
      words[j] = usable ? (uint32_t)half[1] << 16 | (uint32_t)half[0] : none;
    }
  }
}

constexpr int kPitch = kPackFeatures + 2;   // of a column's features in the LDS: the four column groups of a read are 8 (fp32: 16) banks apart

// What a workgroup of the two kernels has: 64 features of an expert, a tile a wave, and every so many-th block of 128 columns.  Workgroups that run at the same time are
// neighbours in the direction that the matrix is contiguous in: columns of [n, k], features of [k, n].
struct PackPlace {
  int n, k, tiles, blocks, feature_groups, experts;
};

// Weights [E, n, k] (TRANSPOSED: [E, k, n]) into words, scales and zeros.  What bounds it: one reading of the weights.  A lane's eight columns of a word
// are 16 bytes in a row of [n, k]; from [k, n] a workgroup's features go through the LDS.  whole: rows are whole 16-byte pieces at 16-byte addresses; the next
// block's are then on their way while a block is encoded.  8 x [14336, 4096] in bf16 as [k, n]: 278 us for 1.18 GB read and written (4.2 TB/s, a copy
// reaches 4.9), back in 225 (5.2 TB/s).
template <int DT, int GROUP, bool TRANSPOSED, bool ZEROS>
__global__ void __launch_bounds__(kPackThreads)
quantize_kernel(const void* __restrict__ weights, const PackPlace place, bool whole, uint32_t* __restrict__ words, void* __restrict__ scales, uint8_t* __restrict__ zeros) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = 16 / sizeof(E), kPieces = kTileColumns * kPackFeatures / kEach / kPackThreads;   // of a thread and block
  __shared__ alignas(16) E staged[TRANSPOSED ? kTileColumns * kPitch : 1];
  const int lane = lane_id(), f = lane % 16, g = lane / 16, n = place.n, k = place.k;
  const int block0 = TRANSPOSED ? blockIdx.y : blockIdx.x, block_step = TRANSPOSED ? gridDim.y : gridDim.x;
  const int group0 = TRANSPOSED ? blockIdx.x : blockIdx.y, group_step = TRANSPOSED ? gridDim.x : gridDim.y;
  for (int64_t expert = blockIdx.z; expert < place.experts; expert += gridDim.z)
    for (int group = group0; group < place.feature_groups; group += group_step) {
      const int first = group * kPackFeatures, tile = group * 4 + (int)(threadIdx.x / kWave), feature = tile * 16 + f;
      const E* const matrix = (const E*)weights + expert * n * k;
      const bool pieces = whole && (!TRANSPOSED || first + kPackFeatures <= n);
      u32x4_t next[kPieces];
      const auto fetch = [&](int block) {
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
          next[q] = u32x4_t{0, 0, 0, 0};
          if constexpr (TRANSPOSED) {
            const int i = q * kPackThreads + (int)threadIdx.x, c = block * kTileColumns + i / (kPackFeatures / kEach);
            if (c < k) next[q] = *(const u32x4_t*)(matrix + (int64_t)c * n + first + i % (kPackFeatures / kEach) * kEach);
          } else {
            const int c = block * kTileColumns + 32 * (q * kEach / 8) + 8 * g + q * kEach % 8;
            if (feature < n && c < k) next[q] = *(const u32x4_t*)(matrix + (int64_t)feature * k + c);
          }
        }
      };
      if (pieces && block0 < place.blocks) fetch(block0);
      for (int block = block0; block < place.blocks; block += block_step) {
        const int column = block * kTileColumns, then = block + block_step;
        float w[4][8];
        if constexpr (TRANSPOSED) {
          __syncthreads();
          if (pieces) {
#pragma unroll
            for (int q = 0; q < kPieces; ++q) {
              const int i = q * kPackThreads + (int)threadIdx.x;
              uint32_t* const to = (uint32_t*)(staged + i / (kPackFeatures / kEach) * kPitch + i % (kPackFeatures / kEach) * kEach);
#pragma unroll
              for (int v = 0; v < 4; ++v) to[v] = next[q][v];
            }
          } else {
            for (int i = threadIdx.x; i < kTileColumns * kPackFeatures; i += kPackThreads) {
              const int c = i / kPackFeatures, r = i % kPackFeatures;
              staged[c * kPitch + r] = column + c < k && first + r < n ? matrix[(int64_t)(column + c) * n + first + r] : E{};
            }
          }
          __syncthreads();
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[j][i] = Elem<DT>::to_f32(staged[(32 * j + 8 * g + i) * kPitch + (tile % 4) * 16 + f]);
        } else if (pieces) {
          E v[4][8];
          __builtin_memcpy(v, next, sizeof(v));
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[j][i] = Elem<DT>::to_f32(v[j][i]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int c = column + 32 * j + 8 * g + i;
              w[j][i] = feature < n && c < k ? Elem<DT>::to_f32(matrix[(int64_t)feature * k + c]) : 0.f;
            }
        }
        if (pieces && then < place.blocks) fetch(then);
        u32x4_t code;
        float scale[kGroups];
        int zero[kGroups];
        encode<DT, GROUP, ZEROS>(w, code, scale, zero);
        if (tile >= place.tiles) continue;   // no barrier between this and the head of the loop, which all waves reach
        const int64_t at = (expert * place.tiles + tile) * place.blocks + block;
        *(u32x4_t*)(words + at * kTileWords + lane * 4) = code;
        // lane 16 q + f has group q's
        float s = scale[0];
        int z = zero[0];
#pragma unroll
        for (int q = 1; q < kGroups; ++q) {
          s = g == q ? scale[q] : s;
          z = g == q ? zero[q] : z;
        }
        if (g < kGroups) {
          ((E*)scales)[at * kGroups * 16 + lane] = Elem<DT>::from_f32(s);
          if constexpr (ZEROS) zeros[at * kGroups * 16 + lane] = (uint8_t)z;
        }
      }
    }
}

// The values: the reverse
template <int DT, int GROUP, bool TRANSPOSED>
__global__ void __launch_bounds__(kPackThreads)
dequantize_kernel(const Packed from, int scale_dtype, const PackPlace place, bool whole, void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  constexpr int kGroups = 128 / GROUP, kEach = 16 / sizeof(E), kPieces = kTileColumns * kPackFeatures / kEach / kPackThreads;
  __shared__ alignas(16) E staged[TRANSPOSED ? kTileColumns * kPitch : 1];
  const int lane = lane_id(), f = lane % 16, g = lane / 16, n = place.n, k = place.k;
  const int block0 = TRANSPOSED ? blockIdx.y : blockIdx.x, block_step = TRANSPOSED ? gridDim.y : gridDim.x;
  const int group0 = TRANSPOSED ? blockIdx.x : blockIdx.y, group_step = TRANSPOSED ? gridDim.x : gridDim.y;
  for (int64_t expert = blockIdx.z; expert < place.experts; expert += gridDim.z)
    for (int group = group0; group < place.feature_groups; group += group_step) {
      const int first = group * kPackFeatures, tile = group * 4 + (int)(threadIdx.x / kWave), feature = tile * 16 + f;
      E* const matrix = (E*)out + expert * n * k;
      const bool pieces = whole && (!TRANSPOSED || first + kPackFeatures <= n);
      u32x4_t code = {0, 0, 0, 0};
      float lane_scale = 0.f, lane_zero = 8.f;    // of group lane / 16 (% the groups)
      const auto fetch = [&](int block) {
        const int64_t at = (expert * place.tiles + tile) * place.blocks + block, i = at * kGroups * 16 + lane % (kGroups * 16);
        code = *(const u32x4_t*)(from.words + at * kTileWords + lane * 4);
        lane_scale = load_as_f32(from.scales, i, scale_dtype);
        if (from.zeros) lane_zero = (float)from.zeros[i];
      };
      if (tile < place.tiles && block0 < place.blocks) fetch(block0);
      for (int block = block0; block < place.blocks; block += block_step) {
        const int column = block * kTileColumns, then = block + block_step;
        uint32_t scale[kGroups], zero[kGroups];
        spread<kGroups>(__float_as_uint(lane_scale), scale);
        spread<kGroups>(__float_as_uint(lane_zero), zero);
        E v[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = __uint_as_float(scale[j * kGroups / 4]), z = __uint_as_float(zero[j * kGroups / 4]);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = Elem<DT>::from_f32(((float)((code[j] >> (4 * (i / 2 + 4 * (i & 1)))) & 15u) - z) * s);
        }
        if (tile < place.tiles && then < place.blocks) fetch(then);
        if constexpr (TRANSPOSED) {
          __syncthreads();
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) staged[(32 * j + 8 * g + i) * kPitch + (tile % 4) * 16 + f] = v[j][i];
          __syncthreads();
          if (pieces) {
#pragma unroll
            for (int q = 0; q < kPieces; ++q) {
              const int i = q * kPackThreads + (int)threadIdx.x, c = i / (kPackFeatures / kEach), r = i % (kPackFeatures / kEach) * kEach;
              const uint32_t* const at = (const uint32_t*)(staged + c * kPitch + r);
              if (column + c < k) *(u32x4_t*)(matrix + (int64_t)(column + c) * n + first + r) = u32x4_t{at[0], at[1], at[2], at[3]};
            }
          } else {
            for (int i = threadIdx.x; i < kTileColumns * kPackFeatures; i += kPackThreads) {
              const int c = i / kPackFeatures, r = i % kPackFeatures;
              if (column + c < k && first + r < n) matrix[(int64_t)(column + c) * n + first + r] = staged[c * kPitch + r];
            }
          }
        } else if (pieces) {
          u32x4_t piece[kPieces];
          __builtin_memcpy(piece, v, sizeof(v));
#pragma unroll
          for (int q = 0; q < kPieces; ++q) {
            const int c = column + 32 * (q * kEach / 8) + 8 * g + q * kEach % 8;
            if (feature < n && c < k) *(u32x4_t*)(matrix + (int64_t)feature * k + c) = piece[q];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int c = column + 32 * j + 8 * g + i;
              if (feature < n && c < k) matrix[(int64_t)feature * k + c] = v[j][i];
            }
        }
      }
    }
}

constexpr int kMostFeatures = 1 << 26;   // a launch's threads have to be fewer than 2^32

static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }

static bool is_dtype(int d) { return d == MBX_BF16 || d == MBX_F16 || d == MBX_F32; }

// Workgroups for all blocks up to 16384 (64 a compute unit), then as many that each has some in turn, up to eight
struct PackGrid {
  PackPlace place;
  dim3 grid;
  PackGrid(int experts, int n, int k, bool transposed) {
    place = {n, k, (int)pieces_of(n, kTileFeatures), (int)pieces_of(k, kTileColumns), (int)pieces_of(n, kPackFeatures), experts};
    const int64_t all = (int64_t)place.blocks * place.feature_groups * experts, turns = pieces_of(all, 16384);
    const int64_t each = turns < 8 ? turns : 8;
    const auto most = [](int64_t v) { return (unsigned)(v < 65535 ? v : 65535); };
    const int64_t columns = pieces_of(place.blocks, (int)each);
    grid = transposed ? dim3((unsigned)place.feature_groups, most(columns), most(experts)) : dim3((unsigned)columns, most(place.feature_groups), most(experts));
  }
};

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

int mbx_quantize_4bit(const void* weights, int dtype, int num_experts, int n, int k, int layout, int group, void* words, void* scales, uint8_t* zeros,
                      mbx_stream_t stream) {
  if (!is_dtype(dtype) || num_experts < 0 || n < 0 || k < 0 || (layout != MBX_NT && layout != MBX_NN) || !group_ok(group)) return MBX_EINVAL;
  if (n > kMostFeatures || k > 0x7fffffff - 256) return MBX_ERANGE;
  if (num_experts == 0 || n == 0 || k == 0) return 0;
  if (!weights || !words || !scales || ((uintptr_t)words & 15)) return MBX_EINVAL;
  const PackGrid p(num_experts, n, k, layout == MBX_NN);
  hipStream_t s = as_stream(stream);
  const int size = dtype_bytes(dtype), row = layout == MBX_NT ? k : n;
  const bool whole = ((uintptr_t)weights & 15) == 0 && row % (16 / size) == 0;
#define MBX_PACK_GROUP(KERNEL, DT, T, ...)                                                      \
  do {                                                                                          \
    if (group == 32) KERNEL(DT, 32, T, __VA_ARGS__);                                            \
    else if (group == 64) KERNEL(DT, 64, T, __VA_ARGS__);                                       \
    else KERNEL(DT, 128, T, __VA_ARGS__);                                                       \
  } while (0)
#define MBX_PACK_TYPE(KERNEL, DT, ...)                                                          \
  do {                                                                                          \
    if (layout == MBX_NN) MBX_PACK_GROUP(KERNEL, DT, true, __VA_ARGS__);                        \
    else MBX_PACK_GROUP(KERNEL, DT, false, __VA_ARGS__);                                        \
  } while (0)
#define MBX_PACK(KERNEL, ...)                                                                   \
  do {                                                                                          \
    if (dtype == MBX_BF16) MBX_PACK_TYPE(KERNEL, MBX_BF16, __VA_ARGS__);                        \
    else if (dtype == MBX_F16) MBX_PACK_TYPE(KERNEL, MBX_F16, __VA_ARGS__);                     \
    else MBX_PACK_TYPE(KERNEL, MBX_F32, __VA_ARGS__);                                           \
  } while (0)
#define MBX_QUANTIZE(DT, GROUP, T, ...)                                                         \
  do {                                                                                          \
    if (zeros) quantize_kernel<DT, GROUP, T, true><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__);  \
    else quantize_kernel<DT, GROUP, T, false><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__);     \
  } while (0)
#define MBX_DEQUANTIZE(DT, GROUP, T, ...) dequantize_kernel<DT, GROUP, T><<<p.grid, kPackThreads, 0, s>>>(__VA_ARGS__)
  MBX_PACK(MBX_QUANTIZE, weights, p.place, whole, (uint32_t*)words, scales, zeros);
  return launch_status();
}

int mbx_dequantize_4bit(const void* words, const void* scales, const uint8_t* zeros, int scale_dtype, int num_experts, int n, int k, int layout, int group,
                        void* out, int dtype, mbx_stream_t stream) {
  if (!is_dtype(dtype) || !is_dtype(scale_dtype) || num_experts < 0 || n < 0 || k < 0 || (layout != MBX_NT && layout != MBX_NN) || !group_ok(group)) return MBX_EINVAL;
  if (n > kMostFeatures || k > 0x7fffffff - 256) return MBX_ERANGE;
  if (num_experts == 0 || n == 0 || k == 0) return 0;
  if (!out || !words || !scales || ((uintptr_t)words & 15)) return MBX_EINVAL;
  const PackGrid p(num_experts, n, k, layout == MBX_NN);
  hipStream_t s = as_stream(stream);
  const int size = dtype_bytes(dtype), row = layout == MBX_NT ? k : n;
  const bool whole = ((uintptr_t)out & 15) == 0 && row % (16 / size) == 0;
  const Packed from = {(const uint32_t*)words, scales, zeros};
  MBX_PACK(MBX_DEQUANTIZE, from, scale_dtype, p.place, whole, out);
#undef MBX_PACK
#undef MBX_PACK_TYPE
#undef MBX_PACK_GROUP
#undef MBX_QUANTIZE
#undef MBX_DEQUANTIZE
  return launch_status();
}

int mbx_gmm_4bit(const void* a, int64_t a_rows, const int32_t* indices, int top_k, const void* words, const void* scales, const uint8_t* zeros,
                 const void* words2, const void* scales2, const uint8_t* zeros2, int scale_dtype, int group, void* c, int dtype, const int32_t* bins,
                 int num_groups, int64_t rows, int k, int n, int act, mbx_stream_t stream) {
  if (!is_dtype(dtype) || !is_dtype(scale_dtype) || !group_ok(group) || num_groups < 0 || rows < 0 || k < 0 || n < 0 || act < -1 || act > MBX_ACT_GELU_TANH) return MBX_EINVAL;
  if (indices && (top_k <= 0 || a_rows < 0)) return MBX_EINVAL;
  if (words2 && (act < 0 || !zeros != !zeros2)) return MBX_EINVAL;
  if (dtype == MBX_F32 || (scale_dtype != dtype && scale_dtype != MBX_F32) || k == 0) return MBX_EUNSUPPORTED;
  if (rows > 0x7fffffff - 64 || n > kMostFeatures || k > 0x7fffffff - 256) return MBX_ERANGE;
  if (rows == 0 || n == 0 || num_groups == 0) return 0;
  if (!a || !words || !scales || !c || !bins || (words2 && !scales2) || (indices && a_rows == 0)) return MBX_EINVAL;
  if (((uintptr_t)words | (uintptr_t)words2) & 15) return MBX_EINVAL;
  hipStream_t s = as_stream(stream);
  const Rows4bit g = {a, indices, a_rows, top_k, {{(const uint32_t*)words, scales, zeros}, {(const uint32_t*)words2, scales2, zeros2}}, scale_dtype == MBX_F32,
                      c, bins, num_groups, rows, k, n, act, 0};
  // By rows an expert in the mean of those that can have some.  The kernel for few goes over the weights again for every 16 rows and has the shorter way, which
  // counts where the weights are few.  Us, of the kernels for few / dozens: 8 gated experts of [4096, 14336], 12 rows 93 / 112, 16 rows 135 / 100; 64 of [2048,
  // 1408], 8 rows 42 / 47, 16 rows 65 / 48; 8 of [14336, 4096] without a gate, 16 rows 75 / 98, 24 rows 95 / 81; 12 of [1032, 2728], 16 rows 16 / 19, 33 rows
  // 24 / 20.  Of those for dozens / hundreds, whose rows are whole pieces of 16 bytes: the first, 64 rows 230 / 239, 128 rows 381 / 345, 1024 rows 2516 / 2030; the
  // second, 93 rows 140 / 138, 384 rows 477 / 405.
  const int64_t experts = rows < num_groups ? rows : num_groups, tiles = pieces_of(n, kTileFeatures) * experts * (words2 ? 2 : 1);
  const bool few = rows <= (tiles <= 4096 ? 20 : 12) * experts, many = rows >= 96 * experts && k % 8 == 0 && k <= 1 << 27;
  const int64_t slots = experts + rows / (few ? 16 : many ? 64 : 32);
  return few ? launch_rows_4bit(g, dtype, group, slots, experts, s) : many ? launch_long_4bit(g, dtype, group, slots, s) : launch_tiles_4bit(g, dtype, group, slots, s);
}

}  // extern "C"
