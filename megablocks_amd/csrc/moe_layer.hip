// A whole mixture-of-experts layer for a few tokens (up to 64), without gradients: the router, the choice of experts, their products, the weighted sum.
//
//   l = x Wr^T;  s = softmax(l) or 1 / (1 + exp(-l));  the top_k experts by key (l, or s + bias; open groups only);  w = scale s / ||s||_p
//   out[t] = sum_j w[t, j] (act(x[t] W1[e]^T) * (x[t] V1[e]^T)) W2[e],  e = the j-th expert of t
//
// What bounds it is reading the weights of the chosen experts, once, and, for a few small ones, the way between the launches.  Three of them:
//
//   choose   a wave per expert and token (or four tokens): logits as exact products summed in 64 bits, so that no order of summation decides between
//            neighbours; the workgroup that is last at a group of tokens chooses for them
//   hidden   a workgroup per used expert and 16 to 128 rows of its first weights, a quarter of the reduction a wave; the activation is kept as two 16-bit
//            numbers, so that the second product sees it to 2^-17 (bf16) or 2^-23 (fp16, or to 2^-32, up to 2^20)
//   down     a workgroup per used expert, 128 columns and a part of the reduction; the parts meet in memory, and the workgroup that is last at its columns adds them up
//            in a fixed order, weights them and writes the output
//
// Measured (us: choose + hidden + down; the weights' rate in the last two, of 5.9 TB/s that a large read reaches):
//    1 token,  6 of 64 gated experts of [1408, 2048]    6.3 +  19 +  12     3.7 and 2.9 TB/s: 528 and 192 workgroups of 5 to 8 chunks a wave, half of it the way to the first
//    1 token,  2 of 8 of [14336, 4096]                  5.1 +  93 +  44     5.1 and 5.3
//    16 tokens, 1 of 64 of [4096, 1024], no gate        6.3 +  24 +  27     4.9 and 4.4
//    5 tokens, 4 of 60 of [2728, 1032], fp16            7.8 +  39 +  27     4.9 and 3.5: rows that begin inside cache lines
//    64 tokens, 2 of 8 of [14336, 4096]                 5.5 + 355 + 183     5.3 and 5.1
//
// "Last" is counted with device-wide atomics; nobody waits for anybody.  What goes from one workgroup to another inside a launch is stored and loaded past the
// caches (the compute units are on eight L2s that do not see each other) and counted in when the stores have been acknowledged.  Sums are taken in an order that
// does not depend on who came when.
#include "gmm_common.h"

#include <cmath>

namespace mbx {
namespace {

constexpr int kLayerTokens = 64, kLayerTopK = 16, kLayerExperts = 512, kLayerGroups = 64;
constexpr int kLayerSlots = kLayerTokens * kLayerTopK;
constexpr int kLayerThreads = 256, kLayerWaves = kLayerThreads / kWave;
constexpr int kLayerMaxParts = 16;                                     // of the second product's reduction
constexpr int kDownColumns = 128;
// counters: from 0 on groups of tokens, then the second product's columns
constexpr int kCounterColumns = kLayerTokens;

struct LayerChoice {
  int tokens, hidden, experts, top_k, sigmoid, groups, top_groups, group_best;
  float norm_p, scale;
};

__device__ __forceinline__ void store_through(uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t load_through(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Whether this workgroup is the last of `all` to come here; what all of them have stored through the caches can then be loaded.  Leaves the counter zero.
__device__ __forceinline__ bool last_to_come(int32_t* counter, int all, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    if (last) *counter = 0;
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

// larger keys first, NaN before all, -0 as 0; 0 is below every number's
__device__ __forceinline__ uint64_t sortable(double key) {
  const uint64_t u = __builtin_bit_cast(uint64_t, key + 0.0);
  return key != key ? ~0ull : (int64_t)u < 0 ? ~u : u | 1ull << 63;
}

// v of all lanes combined, in all of them: wave_butterfly of two registers a value
template <typename F>
__device__ __forceinline__ double wave_butterfly_f64(double v, F&& op) {
  const auto value = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo); };
  const auto low = [](double x) { return (uint32_t)__builtin_bit_cast(uint64_t, x); };
  const auto high = [](double x) { return (uint32_t)(__builtin_bit_cast(uint64_t, x) >> 32); };
  {
    const auto lo = __builtin_amdgcn_permlane32_swap(low(v), low(v), false, false), hi = __builtin_amdgcn_permlane32_swap(high(v), high(v), false, false);
    v = op(value(lo[0], hi[0]), value(lo[1], hi[1]));
  }
  {
    const auto lo = __builtin_amdgcn_permlane16_swap(low(v), low(v), false, false), hi = __builtin_amdgcn_permlane16_swap(high(v), high(v), false, false);
    v = op(value(lo[0], hi[0]), value(lo[1], hi[1]));
  }
  v = op(v, value(lane_xor_dpp<8>(low(v)), lane_xor_dpp<8>(high(v))));
  v = op(v, value(lane_xor_dpp<4>(low(v)), lane_xor_dpp<4>(high(v))));
  v = op(v, value(lane_xor_dpp<2>(low(v)), lane_xor_dpp<2>(high(v))));
  return op(v, value(lane_xor_dpp<1>(low(v)), lane_xor_dpp<1>(high(v))));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  return wave_butterfly_f64(v, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double wave_max_f64(double v) {
  return wave_butterfly_f64(v, [](double a, double b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  return wave_butterfly(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
  return wave_butterfly(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// The choice for a token by one wave: expert 64 i + lane is in register i.  scratch: this wave's, a value for every expert (groups only).
// logit(e): the token's; put(j, e): its j-th expert.
template <int R, typename L, typename P>
__device__ __forceinline__ void choose_for(const LayerChoice& q, int token, L&& logit, const float* __restrict__ bias, double* __restrict__ scratch,
                                           float* __restrict__ weights, int64_t* __restrict__ indices, P&& put) {
  const int lane = lane_id();
  double score[R];
  uint64_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = i * kWave + lane;
    score[i] = e < q.experts ? logit(e) : -INFINITY;
    key[i] = e < q.experts ? sortable(score[i]) : 0;
  }
  if (q.sigmoid) {
#pragma unroll
    for (int i = 0; i < R; ++i) score[i] = 1. / (1. + exp(-score[i]));
  } else {
    double most = -INFINITY, sum = 0.;
#pragma unroll
    for (int i = 0; i < R; ++i) most = score[i] > most ? score[i] : most;
    most = wave_max_f64(most);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      score[i] = exp(score[i] - most);
      sum += i * kWave + lane < q.experts ? score[i] : 0.;
    }
    sum = wave_sum_f64(sum);
#pragma unroll
    for (int i = 0; i < R; ++i) score[i] /= sum;
  }
  if (bias != nullptr) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = i * kWave + lane;
      if (e < q.experts) key[i] = sortable(score[i] + (double)bias[e]);
    }
  }
  if (q.top_groups < q.groups) {
    const int size = q.experts / q.groups;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = i * kWave + lane;
      // without a bias a group that goes by its best expert goes by that one's logit, as the choice does: scores of 1 - 1e-17 are all 1
      if (e < q.experts) scratch[e] = bias != nullptr ? score[i] + (double)bias[e] : q.group_best == 1 ? logit(e) : score[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double best = -INFINITY, second = -INFINITY;
    if (lane < q.groups)
      for (int i = 0; i < size; ++i) {
        const double v = scratch[lane * size + i];
        if (v > best || v != v) { second = best; best = v; }
        else if (v > second) second = v;
      }
    const uint64_t mine = lane < q.groups ? sortable(q.group_best == 2 && size > 1 ? best + second : best) : 0;
    int before = 0;
    for (int g = 0; g < q.groups; ++g) {
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), g) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, g);
      before += other > mine || (other == mine && g < lane) ? 1 : 0;
    }
    const uint64_t open = __ballot(lane < q.groups && before < q.top_groups);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = i * kWave + lane;
      if (e < q.experts && !(open >> (e / size) & 1)) key[i] = 0;
    }
  }
  int my_expert = 0;          // lane j: the j-th of the choice
  double my_score = 0.;
  for (int j = 0; j < q.top_k; ++j) {
    uint64_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < R; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
    const uint32_t high = wave_max_u32((uint32_t)(best >> 32));
    const bool high_is = (uint32_t)(best >> 32) == high;
    const uint64_t tied = __ballot(high_is);
    int e;
    if ((tied & (tied - 1)) == 0) {      // nearly always
      e = __builtin_amdgcn_readlane(at * kWave + lane, __builtin_ctzll(tied));
    } else {
      const uint32_t low = wave_max_u32(high_is ? (uint32_t)best : 0u);
      e = __builtin_amdgcn_readfirstlane((int)wave_min_u32(high_is && (uint32_t)best == low ? (uint32_t)(at * kWave + lane) : ~0u));
    }
    const int from = e % kWave, reg = e / kWave;
    double s = 0.;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i == reg) {
        s = score[i];
        if (lane == from) key[i] = 0;
      }
    const uint64_t bits = __builtin_bit_cast(uint64_t, s);
    s = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)bits, from));
    if (lane == j) {
      my_expert = e;
      my_score = s;
    }
  }
  double weight = my_score;
  if (q.norm_p > 0.f) {
    // the norm as the largest times the norm of the scores over that: scores of 1e-20, or large p, have powers below the smallest number
    const double p = q.norm_p, s = lane < q.top_k ? my_score : 0., most = wave_max_f64(s), part = p != 1. && most > 0. ? s / most : s;
    const double sum = wave_sum_f64(p == 1. ? part : p == 2. ? part * part : pow(part, p));
    weight = sum == 0. ? 0. : part / (p == 1. ? sum : p == 2. ? sqrt(sum) : pow(sum, 1. / p));      // scores that are all zero: weights of zero
  }
  if (lane < q.top_k) {
    const int64_t at = (int64_t)token * q.top_k + lane;
    weights[at] = (float)(weight * (double)q.scale);
    indices[at] = my_expert;
    put(lane, my_expert);
  }
}

// ---- choose ----
// sums of exact products in 64 bits of EB rows of the router and TB tokens, in all lanes
template <int DT, int EB, int TB>
__device__ __forceinline__ void dot_f64(const uint16_t* __restrict__ router, int e0, int experts, const uint16_t* __restrict__ x, int t0, int tokens, int hidden,
                                        double (&acc)[EB][TB]) {
  typedef typename Elem<DT>::type E;
  constexpr int kAhead = EB * TB == 1 ? 8 : 2, kStep = kWave * 8;
#pragma unroll
  for (int e = 0; e < EB; ++e)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[e][t] = 0.;
  for (int c0 = lane_id() * 8; c0 < hidden; c0 += kAhead * kStep) {
    u32x4 w[kAhead][EB], v[kAhead][TB];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u * kStep;
      const bool here = c < hidden;
#pragma unroll
      for (int e = 0; e < EB; ++e) w[u][e] = here && e0 + e < experts ? *(const u32x4*)(router + (int64_t)(e0 + e) * hidden + c) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < TB; ++t) v[u][t] = here && t0 + t < tokens ? *(const u32x4*)(x + (int64_t)(t0 + t) * hidden + c) : u32x4{0u, 0u, 0u, 0u};
    }
    const auto value = [](const u32x4& p, int i) { return (double)Elem<DT>::to_f32(__builtin_bit_cast(E, (uint16_t)(p[i >> 1] >> ((i & 1) * 16)))); };
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        double wd[EB];
#pragma unroll
        for (int e = 0; e < EB; ++e) wd[e] = value(w[u][e], i);
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          const double vd = value(v[u][t], i);
#pragma unroll
          for (int e = 0; e < EB; ++e) acc[e][t] = __builtin_fma(wd[e], vd, acc[e][t]);
        }
      }
  }
#pragma unroll
  for (int e = 0; e < EB; ++e)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[e][t] = wave_sum_f64(acc[e][t]);
}

// A workgroup a token, of sixteen waves: for routers a compute unit reads in the time that the exchange between several takes.
constexpr int kWholeThreads = 1024, kWholeWaves = kWholeThreads / kWave;
template <int DT, int EB, int R>
__global__ void __launch_bounds__(kWholeThreads)
layer_choose_whole_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ router, LayerChoice q, const float* __restrict__ bias, int32_t* __restrict__ choice,
                          float* __restrict__ weights, int64_t* __restrict__ indices) {
  __shared__ double logits[R * kWave], scratch[R * kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), token = blockIdx.x;
  for (int e0 = wave * EB; e0 < q.experts; e0 += kWholeWaves * EB) {
    double acc[EB][1];
    dot_f64<DT, EB, 1>(router, e0, q.experts, x, token, q.tokens, q.hidden, acc);
#pragma unroll
    for (int e = 0; e < EB; ++e)
      if (lane_id() == e && e0 + e < q.experts) logits[e0 + e] = acc[e][0];
  }
  __syncthreads();
  if (wave == 0)
    choose_for<R>(q, token, [&](int e) { return logits[e]; }, bias, scratch, weights, indices, [&](int j, int e) { choice[(int64_t)token * q.top_k + j] = e; });
}

// Workgroup (b, g): experts 4 b .. 4 b + 3, a wave each, tokens TB g .. ; TB 1 or 4.
template <int DT, int TB, int R>
__global__ void __launch_bounds__(kLayerThreads)
layer_choose_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ router, LayerChoice q, const float* __restrict__ bias, uint64_t* __restrict__ logits,
                    int32_t* __restrict__ choice, float* __restrict__ weights, int64_t* __restrict__ indices, int32_t* __restrict__ counters) {
  __shared__ double scratch[kLayerWaves][R * kWave];
  __shared__ int flag;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int e = (int)blockIdx.x * kLayerWaves + wave, t0 = (int)blockIdx.y * TB, tokens = q.tokens - t0 < TB ? q.tokens - t0 : TB;
  if (e < q.experts) {
    double acc[1][TB];
    dot_f64<DT, 1, TB>(router, e, q.experts, x, t0, q.tokens, q.hidden, acc);
#pragma unroll
    for (int t = 0; t < TB; ++t)
      if (lane_id() == t && t < tokens) store_through(logits + (int64_t)(t0 + t) * q.experts + e, __builtin_bit_cast(uint64_t, acc[0][t]));
  }
  if (!last_to_come(counters + blockIdx.y, (int)gridDim.x, &flag)) return;
  for (int t = t0 + wave; t < t0 + tokens; t += kLayerWaves)
    choose_for<R>(q, t, [&](int e) { return __builtin_bit_cast(double, load_through(logits + (int64_t)t * q.experts + e)); }, bias, scratch[wave], weights, indices,
                  [&](int j, int e) { choice[(int64_t)t * q.top_k + j] = e; });
}

// ---- products ----
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if (DT == MBX_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

constexpr uint32_t kNone = 0x80000000u;      // an offset past every buffer: the load brings zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t at) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0)); }

__device__ __forceinline__ float activated(float x, int act) {
  // silu: x / (1 + exp(-x));  gelu: x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
  const float z = act == MBX_ACT_SILU ? x * -1.44269504f : x * (-0.102943240f * (x * x) - 2.30220819f);
  return x / (1.f + __builtin_amdgcn_exp2f(z));
}

// v as unit (hi + rest lo), two 16-bit numbers.  fp16 has no step below 2^-24 and nothing past 65504: what the first number leaves is kept times 2^11, which fits where
// the first does, and both are sixteenths.  So v is kept to 2^-23 of it or 2^-32, up to 2^20.
template <int DT> struct InTwo { static constexpr float unit = DT == MBX_F16 ? 16.f : 1.f, rest = DT == MBX_F16 ? 0x1p-11f : 1.f; };
template <int DT>
__device__ __forceinline__ void in_two(float v, uint16_t& hi, uint16_t& lo) {
  typedef typename Elem<DT>::type E;
  v *= 1.f / InTwo<DT>::unit;
  const E h = Elem<DT>::from_f32(v);
  const float rest = (v - Elem<DT>::to_f32(h)) * (1.f / InTwo<DT>::rest);
  hi = __builtin_bit_cast(uint16_t, h);
  lo = __builtin_bit_cast(uint16_t, Elem<DT>::from_f32(rest - rest == 0.f ? rest : 0.f));     // an infinity or NaN has no rest
}

// The assignments (token top_k + j, one a token at most) of the u-th of the experts that have any, experts and tokens ascending: every workgroup finds them for
// itself out of the choice, 4 KiB at most.  A table of them, made by the workgroup that is the last of all to choose, takes an exchange between workgroups and a way
// to memory more (us a layer with it / so: 16 tokens, 1 of 64 experts of [4096, 1024] 63.5 / 62.3; 64 tokens, 1 of 4 of [1024, 1024] 27.8 / 26.0; 5, 4 of 60 of [2728, 1032] 76.2 / 75.5; but
// 64 tokens, 16 of 256 of [512, 512], 9000 workgroups with little to do, 126 / 134).  A lone token's u-th expert is the u-th of its choice.
struct LayerRows {
  uint64_t used[kLayerExperts / 8];                // a byte an expert
  int16_t slot_of[kLayerTokens];                   // -1: none
  uint16_t slots[kLayerWaves][kLayerTokens];       // every wave's own copy
};
// the u-th used expert; rows: how many it has, all: how many are used; rows 0 where u is past them
__device__ __forceinline__ int find_rows(const int32_t* __restrict__ choice, int tokens, int top_k, int u, LayerRows& of, int& rows, int& all) {
  static_assert(kLayerTokens == kWave && kLayerExperts == 8 * kWave, "a token a lane, eight experts a lane");
  constexpr int kEach = kLayerSlots / kLayerThreads;
  const int slots = tokens * top_k, i = threadIdx.x, lane = lane_id(), wave = i / kWave;
  if (tokens == 1) {
    all = top_k;
    rows = u < top_k ? 1 : 0;
    if (lane == 0) of.slots[wave][0] = (uint16_t)u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return choice[u < top_k ? u : 0];
  }
  int e[kEach];
#pragma unroll
  for (int n = 0; n < kEach; ++n) e[n] = i + n * kLayerThreads < slots ? choice[i + n * kLayerThreads] : -1;
  if (i < kWave) {
    of.used[i] = 0;
    of.slot_of[i] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kEach; ++n)
    if (n * kLayerThreads < slots && e[n] >= 0) ((uint8_t*)of.used)[e[n]] = 1;
  __syncthreads();
  const uint64_t mine = of.used[lane];
  const int count = __popcll(mine), through = wave_inclusive_scan(count);
  all = __builtin_amdgcn_readlane(through, kWave - 1);
  rows = 0;
  if (u >= all) return 0;
  const int at = __builtin_ctzll(__ballot(through > u));
  uint64_t left = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
  for (int before = u - (__builtin_amdgcn_readlane(through, at) - __builtin_amdgcn_readlane(count, at)); before > 0; --before) left &= left - 1;
  const int expert = at * 8 + __builtin_ctzll(left) / 8;
#pragma unroll
  for (int n = 0; n < kEach; ++n)
    if (n * kLayerThreads < slots && e[n] == expert) of.slot_of[(i + n * kLayerThreads) / top_k] = (int16_t)(i + n * kLayerThreads);
  __syncthreads();
  const int slot = of.slot_of[lane];
  const uint64_t has = __ballot(slot >= 0);
  if (slot >= 0) of.slots[wave][__popcll(has & ((1ull << lane) - 1))] = (uint16_t)slot;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  rows = __popcll(has);
  return expert;
}

// NF fragments of 16 weight rows (with the gate: half of them W1's, half V1's), up to R tiles of 16 token rows.  Of a chunk of 64 columns lane (c = l % 16,
// g = l / 16) has columns 8 g .. 8 g + 7 and 32 + 8 g .. 32 + 8 g + 7 of weight row c and of token row c, 16 bytes each: whole 64-byte pieces a load.
template <int DT, bool GATE, int NF, int R>
__global__ void __launch_bounds__(kLayerThreads)
layer_hidden_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w1, const uint16_t* __restrict__ v1, const int32_t* __restrict__ choice, int tokens,
                    int top_k, int hidden, int ffn, int tiles, int act, uint16_t* __restrict__ h_hi, uint16_t* __restrict__ h_lo) {
  constexpr int kCols = GATE ? NF * 8 : NF * 16;          // output columns
  constexpr int kPitch = NF * 16 + 4, kChunk = 64;
  __shared__ __attribute__((aligned(16))) float sums[kLayerWaves][16][kPitch];
  __shared__ LayerRows of;
  const int u = (int)blockIdx.x / tiles, f0 = ((int)blockIdx.x - u * tiles) * kCols;
  int all_rows, used;
  const int expert = find_rows(choice, tokens, top_k, u, of, all_rows, used);
  if (all_rows == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id(), c = lane & 15, g = lane >> 4;
  const uint32_t pitch = (uint32_t)hidden * 2u;
  const int64_t matrix = (int64_t)ffn * hidden;
  const __amdgpu_buffer_rsrc_t rsrc_x = rsrc_of(x, (uint32_t)tokens * pitch), rsrc_w = rsrc_of(w1 + expert * matrix, (uint32_t)(matrix * 2));
  const __amdgpu_buffer_rsrc_t rsrc_v = GATE ? rsrc_of(v1 + expert * matrix, (uint32_t)(matrix * 2)) : rsrc_w;
  for (int done = 0; done < all_rows; done += 16 * R) {      // once, but for experts of many rows
    const int rows = all_rows - done < 16 * R ? all_rows - done : 16 * R, row_tiles = (rows + 15) / 16;
    uint32_t x_off[R];
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const int r = t * 16 + c;
      x_off[t] = r < rows ? (uint32_t)of.slots[wave][done + r] / (uint32_t)top_k * pitch + (uint32_t)g * 16u : kNone;
    }
    const uint32_t w_off = (uint32_t)(f0 + c) * pitch + (uint32_t)g * 16u;
    struct Chunk { u32x4 a[R][2], b[NF][2]; };
    const int chunks = (hidden + kChunk - 1) / kChunk;
    auto fetch = [&](Chunk& q, int chunk) {
      const uint32_t at = (uint32_t)chunk * (kChunk * 2);
      const uint32_t past[2] = {chunk * kChunk + 8 * g < hidden ? 0u : kNone, chunk * kChunk + 8 * g + 32 < hidden ? 0u : kNone};      // pieces past the row's end
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const int row = GATE ? f % (NF / 2 > 0 ? NF / 2 : 1) : f;
          q.b[f][s] = load16(GATE && f >= NF / 2 ? rsrc_v : rsrc_w, (w_off + at + (uint32_t)(row * 16) * pitch + 64u * s) | past[s]);
        }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < R; ++t)
          if (t == 0 || t < row_tiles) q.a[t][s] = load16(rsrc_x, (x_off[t] + at + 64u * s) | past[s] | (x_off[t] & kNone));
    };
    f32x4 acc[R][NF];
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int f = 0; f < NF; ++f) acc[t][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Chunk& q) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < R; ++t)
          if (t == 0 || t < row_tiles)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[t][f] = mfma<DT>(q.b[f][s], q.a[t][s], acc[t][f]);
    };
    // The waves take the chunks in turn, every workgroup from another one on and round: started together at the rows' beginnings they would all ask for bytes that
    // are a power of two apart, of a few memory channels (1 token, 2 of 8 experts of [14336, 4096]: the layer 164 us, now 148).
    const int steps = chunks > wave ? (chunks - wave + kLayerWaves - 1) / kLayerWaves : 0;      // this wave's
    const int turn = steps > 0 ? (int)(((uint32_t)(f0 / kCols) * 5u + (uint32_t)u * 3u) % (uint32_t)steps) : 0;
    auto chunk_of = [&](int step) {
      const int at = step + turn < steps ? step + turn : step + turn - steps;
      return step < steps ? at * kLayerWaves + wave : chunks;      // past the last one nothing is fetched
    };
    Chunk q0, q1;
    fetch(q0, chunk_of(0));
    for (int step = 0; step < steps; step += 2) {
      fetch(q1, chunk_of(step + 1));
      __builtin_amdgcn_sched_barrier(0);      // a chunk's loads are all issued before the products of the one before it
      multiply(q0);
      __builtin_amdgcn_sched_barrier(0);
      fetch(q0, chunk_of(step + 2));
      __builtin_amdgcn_sched_barrier(0);
      multiply(q1);
      __builtin_amdgcn_sched_barrier(0);
    }
    // accumulator t, f, register i of lane (c, g): token row 16 t + c, weight row 16 f + 4 g + i
    constexpr int kEach = kCols / 16;
    const int m = threadIdx.x / 16, col = threadIdx.x % 16 * kEach;
    for (int t = 0; t < row_tiles; ++t) {
      if (t > 0 || done > 0) __syncthreads();
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        f32x4 v = acc[0][f];
#pragma unroll
        for (int o = 1; o < R; ++o)
          if (t == o) v = acc[o][f];
        *(f32x4*)&sums[wave][c][f * 16 + 4 * g] = v;
      }
      __syncthreads();
      const int r = t * 16 + m;
      if (r < rows && f0 + col < ffn) {      // ffn is a multiple of 8, a thread's columns 1, 2, 4 or 8
        uint16_t hi[kEach], lo[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          float v = 0.f, gate = 0.f;
#pragma unroll
          for (int w = 0; w < kLayerWaves; ++w) {
            v += sums[w][m][col + i];
            if (GATE) gate += sums[w][m][kCols + col + i];
          }
          v = activated(v, act);
          in_two<DT>(GATE ? v * gate : v, hi[i], lo[i]);
        }
        const int64_t at = (int64_t)of.slots[wave][done + r] * ffn + f0 + col;
        __builtin_memcpy(h_hi + at, hi, sizeof(hi));
        __builtin_memcpy(h_lo + at, lo, sizeof(lo));
      }
    }
  }
}

// Second product: 128 columns, in chunks of 32 rows of W2.  Lane (c, g) reads columns 8 c .. 8 c + 7 of rows 8 g .. 8 g + 7, 16 bytes each (256 contiguous bytes a
// row), and turns the 8 x 8 values over with byte permutes: fragment j has column 8 c + j of those rows.
template <int DT, int R>
__global__ void __launch_bounds__(kLayerThreads, R == 4 ? 1 : 2)
layer_down_kernel(const uint16_t* __restrict__ h_hi, const uint16_t* __restrict__ h_lo, const uint16_t* __restrict__ w2, const int32_t* __restrict__ choice, int tokens,
                  int top_k, int hidden, int ffn, int tiles, int parts, const float* __restrict__ weights, float* __restrict__ sums_of_parts, uint16_t* __restrict__ out,
                  int32_t* __restrict__ counters, bool by_xcd) {
  constexpr int kPitch = kDownColumns + 4, kChunk = 32, kThrough = 0x11;      // cache policy: past the caches
  __shared__ __attribute__((aligned(16))) float sums[kLayerWaves][16][kPitch];
  __shared__ LayerRows of;
  __shared__ int flag;
  const int in_order = by_xcd ? xcd_tile_id((int)blockIdx.x, tiles) : (int)blockIdx.x, u = in_order / (tiles * parts), in = in_order - u * tiles * parts;
  const int part = in / tiles, tile = in - part * tiles, n0 = tile * kDownColumns;
  int all_rows, used;
  const int expert = find_rows(choice, tokens, top_k, u, of, all_rows, used), slots = tokens * top_k;
  if (all_rows == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id(), c = lane & 15, g = lane >> 4;
  const uint32_t pitch = (uint32_t)hidden * 2u, h_pitch = (uint32_t)ffn * 2u;
  const int64_t matrix = (int64_t)ffn * hidden;
  const __amdgpu_buffer_rsrc_t rsrc_w = rsrc_of(w2 + expert * matrix, (uint32_t)(matrix * 2));
  const __amdgpu_buffer_rsrc_t rsrc_hi = rsrc_of(h_hi, (uint32_t)slots * h_pitch), rsrc_lo = rsrc_of(h_lo, (uint32_t)slots * h_pitch);
  const uint32_t w_off = n0 + 8 * c < hidden ? (uint32_t)(8 * g) * pitch + (uint32_t)(n0 + 8 * c) * 2u : kNone;
  const int m = threadIdx.x / 16, col = threadIdx.x % 16 * 8;
  const bool mine = n0 + col < hidden;          // a multiple of 8
  // a part's sums lie [part][row][column]
  const __amdgpu_buffer_rsrc_t rsrc_parts = rsrc_of(sums_of_parts, (uint32_t)parts * (uint32_t)slots * (uint32_t)hidden * 4u);
  for (int done = 0; done < all_rows; done += 16 * R) {      // once, but for experts of many rows
    const int rows = all_rows - done < 16 * R ? all_rows - done : 16 * R, row_tiles = (rows + 15) / 16;
    uint32_t h_off[R];
#pragma unroll
    for (int t = 0; t < R; ++t) h_off[t] = t * 16 + c < rows ? (uint32_t)of.slots[wave][done + t * 16 + c] * h_pitch + (uint32_t)g * 16u : kNone;
    const int chunks = (ffn + kChunk - 1) / kChunk, begin = (int)((int64_t)part * chunks / parts), end = (int)((int64_t)(part + 1) * chunks / parts);
    struct Chunk { u32x4 hi[R], lo[R], b[8]; };
    auto fetch = [&](Chunk& q, int chunk) {
      const uint32_t none = chunk < end && w_off != kNone ? 0u : kNone;
      const uint32_t at = w_off + (uint32_t)chunk * kChunk * pitch;      // rows past ffn are past the buffer
#pragma unroll
      for (int i = 0; i < 8; ++i) q.b[i] = load16(rsrc_w, (at + (uint32_t)i * pitch) | none);
      const uint32_t past = chunk < end && chunk * kChunk + 8 * g < ffn ? 0u : kNone;
#pragma unroll
      for (int t = 0; t < R; ++t)
        if (t == 0 || t < row_tiles) {
          const uint32_t h_at = (h_off[t] + (uint32_t)chunk * (kChunk * 2)) | past | (h_off[t] & kNone);
          q.hi[t] = load16(rsrc_hi, h_at);
          q.lo[t] = load16(rsrc_lo, h_at);
        }
    };
    f32x4 acc[R][8];
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Chunk& q) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u32x4 b;
#pragma unroll
        for (int w = 0; w < 4; ++w) b[w] = __builtin_amdgcn_perm(q.b[2 * w + 1][j >> 1], q.b[2 * w][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int t = 0; t < R; ++t)
          if (t == 0 || t < row_tiles) {
            acc[t][j] = mfma<DT>(b, q.hi[t], acc[t][j]);
            if constexpr (InTwo<DT>::rest == 1.f) {
              acc[t][j] = mfma<DT>(b, q.lo[t], acc[t][j]);
            } else {
              const f32x4 rest = mfma<DT>(b, q.lo[t], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[t][j][i] = fmaf(rest[i], InTwo<DT>::rest, acc[t][j][i]);
            }
          }
      }
    };
    Chunk q0, q1;
    fetch(q0, begin + wave);
    for (int chunk = begin + wave; chunk < end; chunk += 2 * kLayerWaves) {
      fetch(q1, chunk + kLayerWaves);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q0);
      __builtin_amdgcn_sched_barrier(0);
      fetch(q0, chunk + 2 * kLayerWaves);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q1);
      __builtin_amdgcn_sched_barrier(0);
    }
    // accumulator t, j, register i of lane (c, g): token row 16 t + c, column 8 (4 g + i) + j
    for (int t = 0; t < row_tiles; ++t) {
      if (t > 0 || done > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = acc[0][j][i];
          hi[j] = acc[0][4 + j][i];
#pragma unroll
          for (int o = 1; o < R; ++o)
            if (t == o) {
              lo[j] = acc[o][j][i];
              hi[j] = acc[o][4 + j][i];
            }
        }
        *(f32x4*)&sums[wave][c][8 * (4 * g + i)] = lo;
        *(f32x4*)&sums[wave][c][8 * (4 * g + i) + 4] = hi;
      }
      __syncthreads();
      if (t * 16 + m < rows && mine) {
        f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
        for (int w = 0; w < kLayerWaves; ++w) {
          lo += *(const f32x4*)&sums[w][m][col];
          hi += *(const f32x4*)&sums[w][m][col + 4];
        }
        const uint32_t at = (((uint32_t)part * (uint32_t)slots + (uint32_t)of.slots[wave][done + t * 16 + m]) * (uint32_t)hidden + (uint32_t)(n0 + col)) * 4u;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, lo), rsrc_parts, (int)at, 0, kThrough);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, hi), rsrc_parts, (int)at + 16, 0, kThrough);
      }
    }
  }
  // Then a token's rows are weighted and added up.  Sixteen threads have a column; with few tokens several of them share a token's parts, and add up in order
  // what each has.
  constexpr int kAhead = 8;
  int share = 1;
  while (tokens * share * 2 <= 16) share *= 2;
  const int pieces = top_k * parts, each = (pieces + share - 1) / share, my_share = m % share, stop = (my_share + 1) * each < pieces ? (my_share + 1) * each : pieces;
  uint32_t place[kAhead];
  float w[kAhead];
  auto look_up = [&](int t, int q) {      // where the pieces q .. of token t lie, and their weights
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool here = q + i < stop && t < tokens && mine;
      const int now = here ? q + i : 0, j = now / parts, p = now - j * parts, s = here ? t * top_k + j : 0;
      const uint32_t at = (((uint32_t)p * (uint32_t)slots + (uint32_t)s) * (uint32_t)hidden + (uint32_t)(n0 + col)) * 4u;
      place[i] = here ? at : kNone;
      w[i] = weights[s];
    }
  };
  look_up(m / share, my_share * each);
  if (!last_to_come(counters + kCounterColumns + tile, used * parts, &flag)) return;
  for (int t0 = 0; t0 < tokens; t0 += 16 / share) {
    const int t = t0 + m / share;
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    for (int q = my_share * each; q < stop; q += kAhead) {
      if (t0 > 0 || q != my_share * each) look_up(t, q);
      u32x4 a[kAhead], b[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        a[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc_parts, (int)place[i], 0, kThrough));
        b[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc_parts, (int)place[i] + 16, 0, kThrough));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (q + i < stop) {
          lo += __builtin_bit_cast(f32x4, a[i]) * w[i];
          hi += __builtin_bit_cast(f32x4, b[i]) * w[i];
        }
    }
    if (share > 1) {      // one round: every token has its threads
      *(f32x4*)&sums[0][m][col] = lo;
      *(f32x4*)&sums[0][m][col + 4] = hi;
      __syncthreads();
      if (my_share != 0) return;
      for (int o = 1; o < share; ++o) {
        lo += *(const f32x4*)&sums[0][m + o][col];
        hi += *(const f32x4*)&sums[0][m + o][col + 4];
      }
    }
    if (t < tokens && mine) {
      lo *= InTwo<DT>::unit;
      hi *= InTwo<DT>::unit;
      const u32x4 v = {pack2<DT>(lo[0], lo[1]), pack2<DT>(lo[2], lo[3]), pack2<DT>(hi[0], hi[1]), pack2<DT>(hi[2], hi[3])};
      *(u32x4*)(out + (int64_t)t * hidden + n0 + col) = v;
    }
  }
}

// ---- host ----
struct LayerPlan {
  int entries;              // experts that can have a row
  double used, rows;        // that get one, and how many those get, where tokens choose evenly
  int fragments, hidden_tiles;
  int row_tiles;            // of 16 rows of an expert that a workgroup has at a time: 1, 2, 4
  int down_tiles, parts;
  bool by_xcd;              // the second product's tiles of an expert's part on one XCD
  size_t choice, logits, h_hi, h_lo, sums, total = 0;

  LayerPlan(int tokens, int hidden, int ffn, int experts, int top_k, bool gate) {
    const int slots = tokens * top_k;
    entries = slots < experts ? slots : experts;
    used = fmin(slots, experts * (1. - pow(1. - (double)top_k / experts, tokens)));
    // Fragments of 16 weight rows a workgroup (half of them W1's, half V1's with a gate; us a layer by 2 / 4 / 8 of them).  From 12 rows an expert on the rows
    // are read again by so many workgroups that eight pay: 64 tokens, 2 of 8 experts of [14336, 4096] 608 / 565 / 544, of [8192, 5120] 462 / 458 / 436, but
    // 4 experts of [1024, 1024], which leave most compute units without a workgroup, 28 / 30 / 34.  Below, two: 1 token, 6 of 64 of [1408, 2048] 41 / 47 / 46, 2 of 8
    // of [12288, 5120] 164 / 183 / 198, 16 tokens, 6 of 64 of [1408, 2048] 179 / 186 / 192.  But rows that are 8 KiB apart come faster in
    // fours: 1 token, 2 of 8 of [14336, 4096] 180 / 166 / 169, of [8192, 4096] 92 / 85, 8 tokens, 4 of 32 of [2048, 4096] 217 / 204, where there are workgroups enough: 1 token, 2 of 8 of
    // [2048, 4096] 38 / 43 / 60.  With a gate no others do (those two with rows of 4160 92 / 98 and 203 / 226, of 8192 153 / 167 and 401 / 397 (8 tokens, 2 of 16 of [4096, 8192] 363 / 413), of 12288 225 / 234 and 577 / 633, of 16384
    // 288 / 284 and 781 / 786); without one the larger powers of two do somewhat (1 token, 2 of 4 of [16384, h], 8 tokens, 4 of 32 of [4096, h]: 4096 105 / 103 and 257 / 261, 8192
    // 206 / 201 and 535 / 503, 12288 296 / 295 and 769 / 800, 16384 374 / 364 and 1012 / 1032).  One without a gate,
    // for a few small experts: 1 token, top-1 of 4 of [2048, 512] 14.7 instead of 15.2.
    const int columns = gate ? 8 : 16;
    const auto workgroups = [&](int n) { return used * ceil_div(ffn, n * columns); };
    rows = slots / used;
    const bool in_fours = gate ? hidden == 4096 : hidden >= 4096 && (hidden & (hidden - 1)) == 0;
    fragments = rows >= 12 && workgroups(8) >= 256 ? 8 : in_fours && workgroups(4) >= 512 ? 4 : gate || workgroups(2) >= 512 ? 2 : 1;
    hidden_tiles = (int)ceil_div(ffn, fragments * columns);
    row_tiles = rows < 12 && (tokens <= 16 || rows <= 8) ? 1 : tokens <= 32 || rows <= 20 ? 2 : 4;
    down_tiles = (int)ceil_div(hidden, kDownColumns);
    // Parts of the second product's reduction, as many as make a workgroup for most compute units, of two chunks a wave and more (us a layer by 1 / 2 / 4 / 8 of them:
    // 1 token, 2 of 8 experts of [14336, 4096], 64 workgroups a part, 209 / 177 / 162 / 164; 6 of 64 of [1408, 2048], 96, 43 / 39 / 41 / 45; 8 of 64 of [2048, 7168],
    // 448, 151 / 152 / 156 / 160; 64 tokens, 6 of 64 of [1408, 2048], 1024, 242 / 254 / 274 / 324).
    parts = 1;
    while (parts < kLayerMaxParts && used * down_tiles * parts < 192 && ceil_div(ffn, 32) >= parts * 4 * kLayerWaves) parts *= 2;
    // Where rows begin inside a cache line, neighbouring tiles share one, which XCDs of their own would each fetch (5 tokens, 4 of 60 of [2728, 1032]: 162 MB for
    // 113): a part's tiles to one XCD, where that leaves none without (us the other way / so: this one 79.6 / 76.3; 33 tokens, 6 of 64 of [1416, 2056] 246 / 234).
    by_xcd = hidden % 64 != 0 && used * parts >= 2 * kXcds;
    auto take = [&](size_t bytes) {
      const size_t at = total;
      total += (bytes + 255) & ~(size_t)255;
      return at;
    };
    choice = take((size_t)slots * 4);
    logits = take((size_t)tokens * experts * 8);
    h_hi = take((size_t)slots * ffn * 2);
    h_lo = take((size_t)slots * ffn * 2);
    sums = take((size_t)parts * slots * hidden * 4);
  }
};

// 0, or why not
int layer_sizes(int64_t tokens, int64_t hidden, int64_t ffn, int experts, int top_k) {
  if (tokens < 0 || hidden < 0 || ffn < 0 || experts <= 0 || top_k <= 0 || top_k > experts) return MBX_EINVAL;
  if (tokens > kLayerTokens || top_k > kLayerTopK || experts > kLayerExperts || hidden == 0 || ffn == 0 || hidden % 8 || ffn % 8) return MBX_EUNSUPPORTED;
  // 32-bit offsets into an expert's matrix (and the rows past it that a tile's fragments ask for), into the hidden rows and the parts; a counter for every tile
  if ((ffn + 64) * hidden * 2 >= (int64_t)1 << 31 || (hidden + 64) * ffn * 2 >= (int64_t)1 << 31 || hidden > (int64_t)(kWorkspaceCounters - kCounterColumns) * kDownColumns ||
      tokens * top_k * ffn * 2 >= (int64_t)1 << 31 || tokens * top_k * hidden * 4 * kLayerMaxParts >= (int64_t)1 << 31 || experts * hidden * 2 >= (int64_t)1 << 31)
    return MBX_ERANGE;
  // a launch's threads have to be fewer than 2^32: a workgroup of the first product has 16 rows of an expert's weights or more
  if ((tokens * top_k < experts ? tokens * top_k : experts) * ceil_div(ffn, 16) * kLayerThreads >= (int64_t)1 << 32) return MBX_ERANGE;
  return 0;
}

template <int DT, int R>
void launch_choose(const void* x_, const void* router_, const LayerChoice& q, const float* bias, char* base, const LayerPlan& plan, float* weights, int64_t* indices,
                   int32_t* counters, hipStream_t s) {
  const uint16_t *const x = (const uint16_t*)x_, *const router = (const uint16_t*)router_;
  int32_t* const choice = (int32_t*)(base + plan.choice);
  // up to 128 KiB of router by one workgroup a token (us, that / four experts a workgroup: 1 token, 8 of 4096 5.2 / 7.4; 16, 64 of 1024 7.9 / 9.4; 1, 64 of 2048 10.5 / 6.4; small
  // layers of 1, 16 and 64 tokens at that border, 64 of 1024 16.8 / 16.4, 21.4 / 22.9, 29.6 / 33.9; 32 of 2048 18.7 / 18.3, 24.6 / 25.2, 32 / 34; 16 of 4096 23.5 / 22.2, 29.0 / 28.0,
  // 36 / 36; 8 of 8192 31 / 31, 38 / 38, 50 / 50; and behind it, 64 of 2048 20.8 / 18.4, 27.4 / 27.4, 40 / 43; 32 of 4096 25 / 22, 31 / 30, 42 / 42)
  if constexpr (R == 1)      // up to 64 experts, as such a router has
    if ((int64_t)q.experts * ((q.hidden + 1023) & ~1023) <= 1 << 16) {
      if (q.experts <= kWholeWaves) layer_choose_whole_kernel<DT, 1, R><<<q.tokens, kWholeThreads, 0, s>>>(x, router, q, bias, choice, weights, indices);
      else layer_choose_whole_kernel<DT, 4, R><<<q.tokens, kWholeThreads, 0, s>>>(x, router, q, bias, choice, weights, indices);
      return;
    }
  const unsigned workgroups = (unsigned)ceil_div(q.experts, kLayerWaves);
  // tokens one by one while there are few waves in all (us, one / two / four / eight of them a wave: 19 tokens, 256 experts of 1104 22 / 17 / 14 / 17, 64 tokens, 128 of
  // 4096 26 / 23 / 20 / 24)
  uint64_t* const logits = (uint64_t*)(base + plan.logits);
  if constexpr (R > 1)      // 64 experts of 64 tokens are no more
    if (q.experts * q.tokens > 4096) {
      layer_choose_kernel<DT, 4, R><<<dim3(workgroups, (unsigned)ceil_div(q.tokens, 4)), kLayerThreads, 0, s>>>(x, router, q, bias, logits, choice, weights, indices, counters);
      return;
    }
  layer_choose_kernel<DT, 1, R><<<dim3(workgroups, (unsigned)q.tokens), kLayerThreads, 0, s>>>(x, router, q, bias, logits, choice, weights, indices, counters);
}

template <int DT, int R>
void launch_products(const void* x, const void* w1, const void* v1, const void* w2, const LayerChoice& q, int ffn, int act, char* base, const LayerPlan& plan,
                     const float* weights, void* out, int32_t* counters, hipStream_t s) {
  const int32_t* const choice = (const int32_t*)(base + plan.choice);
  uint16_t *const hi = (uint16_t*)(base + plan.h_hi), *const lo = (uint16_t*)(base + plan.h_lo);
  const unsigned grid = (unsigned)(plan.entries * plan.hidden_tiles);
#define MBX_LAYER_HIDDEN(GATE, NF) \
  layer_hidden_kernel<DT, GATE, NF, R><<<grid, kLayerThreads, 0, s>>>((const uint16_t*)x, (const uint16_t*)w1, (const uint16_t*)v1, choice, q.tokens, q.top_k, q.hidden, ffn, plan.hidden_tiles, act, hi, lo)
  if constexpr (R > 1)      // from 12 rows an expert on
    if (plan.fragments == 8) { if (v1) MBX_LAYER_HIDDEN(true, 8); else MBX_LAYER_HIDDEN(false, 8); }
  if constexpr (R < 4)      // below: where eight are too few workgroups, so are four
    if (plan.fragments == 4) { if (v1) MBX_LAYER_HIDDEN(true, 4); else MBX_LAYER_HIDDEN(false, 4); }
  if (plan.fragments == 2) { if (v1) MBX_LAYER_HIDDEN(true, 2); else MBX_LAYER_HIDDEN(false, 2); }
  else if (plan.fragments == 1) MBX_LAYER_HIDDEN(false, 1);
#undef MBX_LAYER_HIDDEN
  const int64_t down = (int64_t)plan.entries * plan.down_tiles * plan.parts;
  layer_down_kernel<DT, R><<<(unsigned)(plan.by_xcd ? xcd_grid(down, plan.down_tiles) : down), kLayerThreads, 0, s>>>(
      hi, lo, (const uint16_t*)w2, choice, q.tokens, q.top_k, q.hidden, ffn, plan.down_tiles, plan.parts, weights, (float*)(base + plan.sums), (uint16_t*)out, counters,
      plan.by_xcd);
}

template <int DT>
int launch_layer(const void* x, const void* router, const void* w1, const void* v1, const void* w2, const LayerChoice& q, const float* bias, int ffn, int act, void* out,
                 float* weights, int64_t* indices, char* base, const LayerPlan& plan, int32_t* counters, hipStream_t s) {
  if (q.experts <= 64) launch_choose<DT, 1>(x, router, q, bias, base, plan, weights, indices, counters, s);
  else if (q.experts <= 256) launch_choose<DT, 4>(x, router, q, bias, base, plan, weights, indices, counters, s);
  else launch_choose<DT, 8>(x, router, q, bias, base, plan, weights, indices, counters, s);
  if (plan.row_tiles == 1) launch_products<DT, 1>(x, w1, v1, w2, q, ffn, act, base, plan, weights, out, counters, s);
  else if (plan.row_tiles == 2) launch_products<DT, 2>(x, w1, v1, w2, q, ffn, act, base, plan, weights, out, counters, s);
  else launch_products<DT, 4>(x, w1, v1, w2, q, ffn, act, base, plan, weights, out, counters, s);
  return launch_status();
}

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

// For tests: how such a layer is computed -- {fragments, row tiles, parts, by_xcd} of LayerPlan, or why it is not.
int mbx_debug_moe_layer_plan(int64_t tokens, int64_t hidden, int64_t ffn, int num_experts, int top_k, int gate, int* of) {
  if (const int rc = layer_sizes(tokens, hidden, ffn, num_experts, top_k)) return rc;
  const LayerPlan plan((int)tokens, (int)hidden, (int)ffn, num_experts, top_k, gate != 0);
  of[0] = plan.fragments;
  of[1] = plan.row_tiles;
  of[2] = plan.parts;
  of[3] = plan.by_xcd;
  return 0;
}

size_t mbx_moe_layer_scratch_bytes(int64_t tokens, int64_t hidden, int64_t ffn, int num_experts, int top_k, int gate) {
  if (layer_sizes(tokens, hidden, ffn, num_experts, top_k) || tokens == 0) return 0;
  return LayerPlan((int)tokens, (int)hidden, (int)ffn, num_experts, top_k, gate != 0).total;
}

int mbx_moe_layer(const void* x, int64_t tokens, int64_t hidden, int dtype, const void* router, int num_experts, int top_k, int score, const float* bias, int groups,
                  int top_groups, int group_best, float norm_p, float scale, const void* w1, const void* v1, const void* w2, int64_t ffn, int act, void* out, float* weights,
                  int64_t* indices, void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes, mbx_stream_t stream) {
  if (const int rc = layer_sizes(tokens, hidden, ffn, num_experts, top_k)) return rc;
  if ((score != MBX_SCORE_SOFTMAX && score != MBX_SCORE_SIGMOID) || groups <= 0 || num_experts % groups || top_groups <= 0 || top_groups > groups ||
      (group_best != 1 && group_best != 2) || top_k > top_groups * (num_experts / groups) || !(norm_p >= 0.f) || std::isinf(norm_p) || !std::isfinite(scale) ||
      (act != MBX_ACT_SILU && act != MBX_ACT_GELU_TANH))
    return MBX_EINVAL;
  if ((dtype != MBX_BF16 && dtype != MBX_F16) || groups > kLayerGroups) return MBX_EUNSUPPORTED;
  if (tokens == 0) return 0;
  if (!x || !router || !w1 || !w2 || !out || !weights || !indices) return MBX_EINVAL;
  if (((uintptr_t)x | (uintptr_t)router | (uintptr_t)w1 | (uintptr_t)v1 | (uintptr_t)w2 | (uintptr_t)out) & 15) return MBX_EUNSUPPORTED;
  const LayerPlan plan((int)tokens, (int)hidden, (int)ffn, num_experts, top_k, v1 != nullptr);
  if (!scratch || scratch_bytes < plan.total || ((uintptr_t)scratch & 15)) return MBX_ESCRATCH;
  if (!workspace || workspace_bytes < kWorkspaceCounters * sizeof(int32_t) || ((uintptr_t)workspace & 3)) return MBX_ESCRATCH;
  const LayerChoice q{(int)tokens, (int)hidden, num_experts, top_k, score == MBX_SCORE_SIGMOID, groups, top_groups, group_best, norm_p, scale};
  hipStream_t s = as_stream(stream);
  return dtype == MBX_BF16 ? launch_layer<MBX_BF16>(x, router, w1, v1, w2, q, bias, (int)ffn, act, out, weights, indices, (char*)scratch, plan, (int32_t*)workspace, s)
                           : launch_layer<MBX_F16>(x, router, w1, v1, w2, q, bias, (int)ffn, act, out, weights, indices, (char*)scratch, plan, (int32_t*)workspace, s);
}

}  // extern "C"
