// The norm of many tensors together, and the tensors times min(1, most / (norm + 1e-6)).
//
//   norm = (sum |g|^p)^(1/p) for p = 1, 2; max |g| for p = inf
//
// A sum over the gradients of a model has 10^9 terms: it is held in 64 bits from the first element on, so neither the squares of large values nor the
// last of many small ones are lost, and a square of a 16-bit or 32-bit value is exact in it.  Every workgroup adds a fixed run of chunks and writes one
// partial sum; those are added in a fixed order, so a norm is the same from run to run.  No atomics, nothing to clear.
//
// What bounds both passes is memory: a conversion and a multiply-add in 64 bits an element are a tenth of what the compute units issue meanwhile.  The second
// pass goes through the tensors from behind: what the first one read last is still in the 256 MiB cache.
//
// Measured: the norm of 554 M bf16 values, 1.1 GB, 187 us + 4.5 for the join (5.9 TB/s); clipped into 554 M fp32 ones 234 (what is left of the last pass's output in the
// cache is written meanwhile) + 663 (3.3 GB, 5.0 TB/s, a copy's rate; with stores past the cache 820); 0.55 GB in place that is short enough 95 + 4.6; 300 tensors of
// 2 M values in all 6.2 and 6.9 a launch, of which there are three each way.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace mbx {
namespace {

constexpr int kNormThreads = 256, kNormTensors = 128, kNormBlocks = 2048;
constexpr int kNormUnroll = 4;                                           // pieces of eight elements a thread has under way
constexpr int64_t kNormChunk = (int64_t)kNormThreads * 8 * kNormUnroll * 2;   // elements: 16384

enum { kNormTwo = 0, kNormOne = 1, kNormInf = 2 };

// what a launch goes through: chunk c of the launch belongs to the last tensor whose first chunk is <= c
struct NormList {
  const void* in[kNormTensors];
  void* out[kNormTensors];
  int64_t numel[kNormTensors];
  int32_t first[kNormTensors];
  uint8_t in_type[kNormTensors], out_type[kNormTensors];
  int32_t tensors, chunks;
};
static_assert(sizeof(NormList) + 64 <= 4096, "kernel arguments");

typedef uint32_t u32x4n __attribute__((ext_vector_type(4)));
// tensors may start anywhere their elements may: the memory unit takes 16-byte accesses at any address
typedef u32x4n __attribute__((aligned(2))) u32x4_at2;
typedef u32x4n __attribute__((aligned(4))) u32x4_at4;

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&v)[8]) {
  if constexpr (DT == MBX_F32) {
    const u32x4n a = *(const u32x4_at4*)((const float*)base + i), b = *(const u32x4_at4*)((const float*)base + i + 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) { v[t] = __uint_as_float(a[t]); v[4 + t] = __uint_as_float(b[t]); }
  } else {
    const u32x4n a = *(const u32x4_at2*)((const uint16_t*)base + i);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      v[t] = Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(a[t >> 1] >> ((t & 1) * 16))));
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t i, const float (&v)[8]) {
  if constexpr (DT == MBX_F32) {
    u32x4n a, b;
#pragma unroll
    for (int t = 0; t < 4; ++t) { a[t] = __float_as_uint(v[t]); b[t] = __float_as_uint(v[4 + t]); }
    *(u32x4_at4*)((float*)base + i) = a;
    *(u32x4_at4*)((float*)base + i + 4) = b;
  } else {
    u32x4n a;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      a[t] = (uint32_t)__builtin_bit_cast(uint16_t, Elem<DT>::from_f32(v[2 * t])) | (uint32_t)__builtin_bit_cast(uint16_t, Elem<DT>::from_f32(v[2 * t + 1])) << 16;
    *(u32x4_at2*)((uint16_t*)base + i) = a;
  }
}

// the larger one, a NaN before all
__device__ __forceinline__ double larger(double m, double a) { return a > m || a != a ? a : m; }

template <int MODE>
__device__ __forceinline__ double joined(double a, double b) { return MODE == kNormInf ? larger(a, b) : a + b; }

template <int MODE>
__device__ __forceinline__ void take(double& acc, float v) {
  if constexpr (MODE == kNormTwo) acc = __builtin_fma((double)v, (double)v, acc);
  else if constexpr (MODE == kNormOne) acc += (double)fabsf(v);
  else acc = larger(acc, (double)fabsf(v));
}

// The workgroup's value, in thread 0 (all of them where `all`).
template <int MODE>
__device__ __forceinline__ double block_join(double v, bool all) {
  __shared__ double waves[kNormThreads / kWave];
#pragma unroll
  for (int off = 32; off; off >>= 1) v = joined<MODE>(v, __shfl_xor(v, off, kWave));
  if (lane_id() == 0) waves[threadIdx.x / kWave] = v;
  __syncthreads();
  double r = 0.;
  if (all || threadIdx.x == 0)
#pragma unroll
    for (int w = 0; w < kNormThreads / kWave; ++w) r = joined<MODE>(r, waves[w]);
  return r;
}

// the tensor that chunk c is in
__device__ __forceinline__ int tensor_of(const NormList& list, int c) {
  int lo = 0, hi = list.tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (list.first[mid] <= c) lo = mid; else hi = mid;
  }
  return lo;
}

template <int DT, int MODE>
__device__ __forceinline__ void chunk_join(const void* base, int64_t begin, int64_t end, double (&acc)[4]) {
  constexpr int64_t kStep = (int64_t)kNormThreads * 8;
  int64_t i = begin + (int64_t)threadIdx.x * 8;
  for (; i + (kNormUnroll - 1) * kStep + 8 <= end; i += kNormUnroll * kStep) {
    float v[kNormUnroll][8];
#pragma unroll
    for (int u = 0; u < kNormUnroll; ++u) load8<DT>(base, i + u * kStep, v[u]);
#pragma unroll
    for (int u = 0; u < kNormUnroll; ++u)
#pragma unroll
      for (int t = 0; t < 8; ++t) take<MODE>(acc[t & 3], v[u][t]);
  }
  for (; i < end; i += kStep) {
    if (i + 8 <= end) {
      float v[8];
      load8<DT>(base, i, v);
#pragma unroll
      for (int t = 0; t < 8; ++t) take<MODE>(acc[t & 3], v[t]);
    } else {
      for (int64_t j = i; j < end; ++j) take<MODE>(acc[0], Elem<DT>::to_f32(((const typename Elem<DT>::type*)base)[j]));
    }
  }
}

// Workgroup b of B adds the chunks [b C / B, (b + 1) C / B) into partials[b].
template <int MODE>
__global__ void __launch_bounds__(kNormThreads) norm_partials_kernel(const NormList list, double* __restrict__ partials) {
  const int begin = (int)((int64_t)blockIdx.x * list.chunks / gridDim.x), end = (int)((int64_t)(blockIdx.x + 1) * list.chunks / gridDim.x);
  double acc[4] = {0., 0., 0., 0.};
  int t = tensor_of(list, begin);
  for (int c = begin; c < end; ++c) {
    while (t + 1 < list.tensors && list.first[t + 1] <= c) ++t;
    const int64_t from = (int64_t)(c - list.first[t]) * kNormChunk, to = from + kNormChunk < list.numel[t] ? from + kNormChunk : list.numel[t];
    switch (list.in_type[t]) {
      case MBX_BF16: chunk_join<MBX_BF16, MODE>(list.in[t], from, to, acc); break;
      case MBX_F16: chunk_join<MBX_F16, MODE>(list.in[t], from, to, acc); break;
      default: chunk_join<MBX_F32, MODE>(list.in[t], from, to, acc);
    }
  }
  const double v = block_join<MODE>(joined<MODE>(joined<MODE>(acc[0], acc[1]), joined<MODE>(acc[2], acc[3])), false);
  if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

// All partial sums joined, in every thread, and the norm they make.
template <int MODE>
__device__ __forceinline__ float norm_of(const double* __restrict__ partials, int count) {
  double v = 0.;
  for (int i = threadIdx.x; i < count; i += kNormThreads) v = joined<MODE>(v, partials[i]);
  v = block_join<MODE>(v, true);
  return (float)(MODE == kNormTwo ? sqrt(v) : v);
}

template <int MODE>
__global__ void __launch_bounds__(kNormThreads) norm_join_kernel(const double* __restrict__ partials, int count, float* __restrict__ norm) {
  const float n = norm_of<MODE>(partials, count);
  if (threadIdx.x == 0) *norm = n;
}

template <int IN, int OUT>
__device__ __forceinline__ void chunk_scale(const void* in, void* out, int64_t begin, int64_t end, float by) {
  constexpr int64_t kStep = (int64_t)kNormThreads * 8;
  int64_t i = begin + (int64_t)threadIdx.x * 8;
  for (; i + (kNormUnroll - 1) * kStep + 8 <= end; i += kNormUnroll * kStep) {
    float v[kNormUnroll][8];
#pragma unroll
    for (int u = 0; u < kNormUnroll; ++u) load8<IN>(in, i + u * kStep, v[u]);
#pragma unroll
    for (int u = 0; u < kNormUnroll; ++u) {
#pragma unroll
      for (int t = 0; t < 8; ++t) v[u][t] *= by;
      store8<OUT>(out, i + u * kStep, v[u]);
    }
  }
  for (; i < end; i += kStep) {
    if (i + 8 <= end) {
      float v[8];
      load8<IN>(in, i, v);
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] *= by;
      store8<OUT>(out, i, v);
    } else {
      for (int64_t j = i; j < end; ++j)
        ((typename Elem<OUT>::type*)out)[j] = Elem<OUT>::from_f32(Elem<IN>::to_f32(((const typename Elem<IN>::type*)in)[j]) * by);
    }
  }
}

// Every workgroup makes the norm out of the partial sums for itself.  Tensors that stay where they are and are short enough are done then.
template <int MODE, bool IN_PLACE>
__global__ void __launch_bounds__(kNormThreads) clip_kernel(const NormList list, const double* __restrict__ partials, int count, float most,
                                                            float* __restrict__ norm) {
  const float n = norm_of<MODE>(partials, count);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  float by = most / (n + 1e-6f);
  by = by > 1.f ? 1.f : by;      // a NaN stays one
  if (IN_PLACE && by == 1.f) return;
  const int block = (int)(gridDim.x - 1 - blockIdx.x);
  const int begin = (int)((int64_t)block * list.chunks / gridDim.x), end = (int)((int64_t)(block + 1) * list.chunks / gridDim.x);
  if (begin == end) return;
  int t = tensor_of(list, end - 1);
  for (int c = end - 1; c >= begin; --c) {
    while (list.first[t] > c) --t;
    const int64_t from = (int64_t)(c - list.first[t]) * kNormChunk, to = from + kNormChunk < list.numel[t] ? from + kNormChunk : list.numel[t];
    const void* const in = list.in[t];
    void* const out = list.out[t];
    switch (list.in_type[t] * 3 + list.out_type[t]) {
      case MBX_BF16 * 3 + MBX_BF16: chunk_scale<MBX_BF16, MBX_BF16>(in, out, from, to, by); break;
      case MBX_BF16 * 3 + MBX_F16: chunk_scale<MBX_BF16, MBX_F16>(in, out, from, to, by); break;
      case MBX_BF16 * 3 + MBX_F32: chunk_scale<MBX_BF16, MBX_F32>(in, out, from, to, by); break;
      case MBX_F16 * 3 + MBX_BF16: chunk_scale<MBX_F16, MBX_BF16>(in, out, from, to, by); break;
      case MBX_F16 * 3 + MBX_F16: chunk_scale<MBX_F16, MBX_F16>(in, out, from, to, by); break;
      case MBX_F16 * 3 + MBX_F32: chunk_scale<MBX_F16, MBX_F32>(in, out, from, to, by); break;
      case MBX_F32 * 3 + MBX_BF16: chunk_scale<MBX_F32, MBX_BF16>(in, out, from, to, by); break;
      case MBX_F32 * 3 + MBX_F16: chunk_scale<MBX_F32, MBX_F16>(in, out, from, to, by); break;
      default: chunk_scale<MBX_F32, MBX_F32>(in, out, from, to, by);
    }
  }
}

// ---- host ----

// The tensors that have elements, in launches of up to kNormTensors of them, with as many workgroups each as their share of the chunks.
struct NormLaunches {
  struct One { int first, count, chunks, blocks; };
  std::vector<int> which;     // tensors with elements
  std::vector<One> all;
  int blocks = 0;

  // a negative code, or 0
  int make(const void* const* in, const int64_t* numel, const int* types, int tensors) {
    int64_t total = 0;
    for (int i = 0; i < tensors; ++i) {
      if (numel[i] < 0 || types[i] < MBX_BF16 || types[i] > MBX_F32 || (numel[i] > 0 && !in[i])) return MBX_EINVAL;
      if (numel[i] == 0) continue;
      which.push_back(i);
      total += ceil_div(numel[i], kNormChunk);
      if (total > 0x7fffffff) return MBX_ERANGE;
    }
    for (size_t first = 0; first < which.size(); first += kNormTensors) {
      One one{(int)first, (int)std::min<size_t>(kNormTensors, which.size() - first), 0, 0};
      for (int i = 0; i < one.count; ++i) one.chunks += (int)ceil_div(numel[which[first + i]], kNormChunk);
      one.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(one.chunks, (int64_t)kNormBlocks * one.chunks / total));
      // a few chunks each: as many to all of them (2934 chunks, 48 M fp32 values into others, by 2048 workgroups 141 us, by 1467 123)
      if (one.chunks < 8 * one.blocks) one.blocks = (int)ceil_div(one.chunks, ceil_div(one.chunks, one.blocks));
      blocks += one.blocks;
      all.push_back(one);
    }
    return 0;
  }

  void fill(const One& one, NormList& list, const void* const* in, void* const* out, const int64_t* numel, const int* types, const int* out_types) const {
    list.tensors = one.count;
    list.chunks = 0;
    for (int i = 0; i < one.count; ++i) {
      const int t = which[one.first + i];
      list.in[i] = in[t];
      list.out[i] = out ? out[t] : nullptr;
      list.numel[i] = numel[t];
      list.in_type[i] = (uint8_t)types[t];
      list.out_type[i] = (uint8_t)(out_types ? out_types[t] : 0);
      list.first[i] = list.chunks;
      list.chunks += (int)ceil_div(numel[t], kNormChunk);
    }
  }
};

// Whether an output lies over another one, or over an input that is not its own in the same place and type.
bool outputs_clash(const void* const* in, void* const* out, const int64_t* numel, const int* types, const int* out_types, const std::vector<int>& which) {
  struct Range { uintptr_t from, to; int tensor; };
  std::vector<Range> ranges;
  ranges.reserve(which.size());
  for (const int t : which) ranges.push_back({(uintptr_t)out[t], (uintptr_t)out[t] + (uintptr_t)numel[t] * dtype_bytes(out_types[t]), t});
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i].from < ranges[i - 1].to) return true;
  for (const int t : which) {
    const uintptr_t from = (uintptr_t)in[t], to = from + (uintptr_t)numel[t] * dtype_bytes(types[t]);
    // the first range that ends behind `from`
    auto r = std::upper_bound(ranges.begin(), ranges.end(), from, [](uintptr_t at, const Range& x) { return at < x.to; });
    for (; r != ranges.end() && r->from < to; ++r)
      if (r->tensor != t || r->from != from || types[t] != out_types[t]) return true;
  }
  return false;
}

template <int MODE>
int launch_partials(const NormLaunches& launches, const void* const* in, const int64_t* numel, const int* types, double* partials, hipStream_t s) {
  NormList list;
  for (const auto& one : launches.all) {
    launches.fill(one, list, in, nullptr, numel, types, nullptr);
    norm_partials_kernel<MODE><<<one.blocks, kNormThreads, 0, s>>>(list, partials);
    partials += one.blocks;
  }
  return launch_status();
}

template <int MODE>
int run_norm(const NormLaunches& launches, const void* const* in, const int64_t* numel, const int* types, double* partials, float* norm, hipStream_t s) {
  const int rc = launch_partials<MODE>(launches, in, numel, types, partials, s);
  if (rc) return rc;
  norm_join_kernel<MODE><<<1, kNormThreads, 0, s>>>(partials, launches.blocks, norm);
  return launch_status();
}

template <int MODE>
int run_clip(const NormLaunches& launches, const void* const* in, void* const* out, const int64_t* numel, const int* types, const int* out_types, bool in_place,
             float most, double* partials, float* norm, hipStream_t s) {
  int rc = launch_partials<MODE>(launches, in, numel, types, partials, s);
  if (rc) return rc;
  NormList list;
  for (size_t l = launches.all.size(); l-- > 0;) {
    const auto& one = launches.all[l];
    launches.fill(one, list, in, out, numel, types, out_types);
    float* const to = l == 0 ? norm : nullptr;
    if (in_place) clip_kernel<MODE, true><<<one.blocks, kNormThreads, 0, s>>>(list, partials, launches.blocks, most, to);
    else clip_kernel<MODE, false><<<one.blocks, kNormThreads, 0, s>>>(list, partials, launches.blocks, most, to);
  }
  return launch_status();
}

int mode_of(float p) { return p == 2.f ? kNormTwo : p == 1.f ? kNormOne : std::isinf(p) && p > 0 ? kNormInf : -1; }

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

size_t mbx_global_norm_scratch_bytes(int tensors) {
  // a workgroup more than kNormBlocks for every launch whose share of them rounds to none
  return tensors <= 0 ? 0 : (size_t)(kNormBlocks + ceil_div(tensors, kNormTensors)) * sizeof(double);
}

int mbx_global_norm(const void* const* tensors, const int64_t* numel, const int* dtypes, int count, float p, float* norm, void* scratch, size_t scratch_bytes,
                    mbx_stream_t stream) try {
  const int mode = mode_of(p);
  if (count < 0 || mode < 0 || !norm || (count > 0 && (!tensors || !numel || !dtypes))) return MBX_EINVAL;
  NormLaunches launches;
  if (const int rc = launches.make(tensors, numel, dtypes, count)) return rc;
  if (launches.blocks > 0 && (!scratch || ((uintptr_t)scratch & 7) || scratch_bytes < (size_t)launches.blocks * sizeof(double))) return MBX_ESCRATCH;
  hipStream_t s = as_stream(stream);
  double* const partials = (double*)scratch;
  if (mode == kNormTwo) return run_norm<kNormTwo>(launches, tensors, numel, dtypes, partials, norm, s);
  if (mode == kNormOne) return run_norm<kNormOne>(launches, tensors, numel, dtypes, partials, norm, s);
  return run_norm<kNormInf>(launches, tensors, numel, dtypes, partials, norm, s);
} catch (...) {
  return MBX_EINVAL;
}

int mbx_clip_by_global_norm(const void* const* tensors, void* const* out, const int64_t* numel, const int* dtypes, const int* out_dtypes, int count, float p,
                            float most, float* norm, void* scratch, size_t scratch_bytes, mbx_stream_t stream) try {
  const int mode = mode_of(p);
  if (count < 0 || mode < 0 || !(most >= 0.f) || !norm || (count > 0 && (!tensors || !out || !numel || !dtypes || !out_dtypes))) return MBX_EINVAL;
  NormLaunches launches;
  if (const int rc = launches.make(tensors, numel, dtypes, count)) return rc;
  bool in_place = true;
  for (const int t : launches.which) {
    if (!out[t] || out_dtypes[t] < MBX_BF16 || out_dtypes[t] > MBX_F32) return MBX_EINVAL;
    in_place = in_place && out[t] == tensors[t] && out_dtypes[t] == dtypes[t];
  }
  if (outputs_clash(tensors, out, numel, dtypes, out_dtypes, launches.which)) return MBX_EINVAL;
  if (launches.blocks > 0 && (!scratch || ((uintptr_t)scratch & 7) || scratch_bytes < (size_t)launches.blocks * sizeof(double))) return MBX_ESCRATCH;
  hipStream_t s = as_stream(stream);
  double* const partials = (double*)scratch;
  if (launches.which.empty()) return run_norm<kNormTwo>(launches, tensors, numel, dtypes, partials, norm, s);    // the norm of nothing is 0
  if (mode == kNormTwo) return run_clip<kNormTwo>(launches, tensors, out, numel, dtypes, out_dtypes, in_place, most, partials, norm, s);
  if (mode == kNormOne) return run_clip<kNormOne>(launches, tensors, out, numel, dtypes, out_dtypes, in_place, most, partials, norm, s);
  return run_clip<kNormInf>(launches, tensors, out, numel, dtypes, out_dtypes, in_place, most, partials, norm, s);
} catch (...) {
  return MBX_EINVAL;
}

}  // extern "C"
