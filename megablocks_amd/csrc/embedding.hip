// Rows of a table by token, times a scale, and the gradient of the table.
//
//   out[i] = scale table[ids[i]]           dtable[v] = scale sum over {i : ids[i] = v} of dout[i], i ascending
//
// Both are bound by memory: the rows read and written once, for the gradient the whole table written, most of it zeros.  The gradient's sums are fp32 (64 bits for
// an fp32 table) in a fixed order: rows are added along the tokens sorted by word (stably), a piece of 32 of them by a wave, whose runs of one word go straight to the table; what a run of
// more than 32 tokens leaves in each of its pieces is kept as it is and added up, in order, by a launch of its own.  So a word that is half of the text costs no more
// than any other, and sums do not depend on timing.
//
// Measured (us): 32767 tokens, two fifths of them padding, 100000 words of 2040 in fp16: rows 52 (268 MB, 5.2 TB/s; a copy moves 4.8), gradient 12.8 sorting, 99 sums and
// zeros (0.49 GB, 5.0 TB/s; a fill writes 6.7), 7 joining.  16384 tokens, 50000 words of 1024 in bf16: 13.1 (5.1 TB/s) and 10.8 + 25.9 (136 MB, 5.3 TB/s) + 4.1.  16 tokens: 2.5.
//
// Sorting: workgroup w owns a range of words and goes through all tokens, counts those of smaller words and lists its own, in order, in LDS: no exchange between
// workgroups, one launch.  Its time is latencies: of the loads, four of which are under way in a wave, and of the claims of places.
//
// A token outside the table gives a row of zeros and no gradient.  Tensors may start anywhere and rows have any length: the memory unit takes 16-byte
// accesses at any address.
#include "common.h"

#include <cmath>
#include <type_traits>

namespace mbx {
namespace {

typedef uint32_t u32x4e __attribute__((ext_vector_type(4)));
typedef u32x4e __attribute__((aligned(2))) u32x4_at2;
typedef u32x4e __attribute__((aligned(4))) u32x4_at4;

constexpr int kEmbThreads = 256, kEmbWaves = kEmbThreads / kWave;
constexpr int kPer = 8;                               // columns of a lane
constexpr int kSlice = kPer * kWave;                  // columns of a wave
constexpr int64_t kEmbMaxBlocks = 1 << 23;            // of a launch, whose threads have to be fewer than 2^32

// kPer values as they lie in memory
template <int DT>
struct Piece {
  u32x4e part[DT == MBX_F32 ? 2 : 1];

  __device__ __forceinline__ void load(const void* at) {
    if constexpr (DT == MBX_F32) {
      part[0] = *(const u32x4_at4*)at;
      part[1] = *(const u32x4_at4*)((const float*)at + 4);
    } else {
      part[0] = *(const u32x4_at2*)at;
    }
  }
  __device__ __forceinline__ float value(int t) const {
    if constexpr (DT == MBX_F32) return __uint_as_float(part[t >> 2][t & 3]);
    else return Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(part[0][t >> 1] >> ((t & 1) * 16))));
  }
};

template <int DT>
__device__ __forceinline__ void store8(void* at, const float (&v)[kPer]) {
  if constexpr (DT == MBX_F32) {
    u32x4e a, b;
#pragma unroll
    for (int t = 0; t < 4; ++t) { a[t] = __float_as_uint(v[t]); b[t] = __float_as_uint(v[4 + t]); }
    *(u32x4_at4*)at = a;
    *(u32x4_at4*)((float*)at + 4) = b;
  } else {
    u32x4e a;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      a[t] = (uint32_t)__builtin_bit_cast(uint16_t, Elem<DT>::from_f32(v[2 * t])) | (uint32_t)__builtin_bit_cast(uint16_t, Elem<DT>::from_f32(v[2 * t + 1])) << 16;
    *(u32x4_at2*)at = a;
  }
}

// What gradients are added up in: where the result has 24 bits, thousands of sums in 24 would be off by several of its last.  It is bound by memory either way (us a pass,
// fp32 / 64 bits: 16384 tokens, 50000 words of 1024 101 / 101; 32767, two fifths of them padding, 49999 of 2040 231 / 240, of which 17 MB are the wider sums of cut runs).
template <int DT> using Sum = std::conditional_t<DT == MBX_F32, double, float>;

// N sums as they lie in memory
template <int N, typename S>
struct Sums {
  typedef S vector __attribute__((ext_vector_type(16 / sizeof(S)), aligned(sizeof(S))));
  static constexpr int kEach = 16 / sizeof(S);
  vector part[N / kEach];

  __device__ __forceinline__ void load(const S* at) {
#pragma unroll
    for (int i = 0; i < N / kEach; ++i) part[i] = *(const vector*)(at + i * kEach);
  }
  __device__ __forceinline__ void store(S* at) const {
#pragma unroll
    for (int i = 0; i < N / kEach; ++i) *(vector*)(at + i * kEach) = part[i];
  }
  __device__ __forceinline__ S value(int t) const { return part[t / kEach][t % kEach]; }
};

// up to kPer columns from `at`, of which `left` are the row's
template <int DT>
__device__ __forceinline__ void load_columns(const void* at, int left, float (&v)[kPer]) {
  if (left >= kPer) {
    Piece<DT> piece;
    piece.load(at);
#pragma unroll
    for (int t = 0; t < kPer; ++t) v[t] = piece.value(t);
  } else {
#pragma unroll
    for (int t = 0; t < kPer; ++t) v[t] = t < left ? Elem<DT>::to_f32(((const typename Elem<DT>::type*)at)[t]) : 0.f;
  }
}

template <int DT>
__device__ __forceinline__ void store_columns(void* at, int left, const float (&v)[kPer]) {
  if (left >= kPer) {
    store8<DT>(at, v);
  } else {
#pragma unroll
    for (int t = 0; t < kPer; ++t)
      if (t < left) ((typename Elem<DT>::type*)at)[t] = Elem<DT>::from_f32(v[t]);
  }
}

// token i, or -1 where it is outside the table
template <typename I>
__device__ __forceinline__ int word_of(const I* __restrict__ ids, int64_t i, int words) {
  const I id = ids[i];
  return id >= 0 && id < (I)words ? (int)id : -1;
}

// ---- out[i] = scale table[ids[i]]: a wave per row and slice of kSlice columns ----
template <int DT, typename I>
__global__ void __launch_bounds__(kEmbThreads) embedding_kernel(const I* __restrict__ ids, int64_t tokens, const void* __restrict__ table, int words, int hidden,
                                                                int slices, float scale, void* __restrict__ out, int64_t first_block) {
  typedef typename Elem<DT>::type E;
  const int64_t unit = (first_block + blockIdx.x) * kEmbWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t i = unit / slices;
  if (i >= tokens) return;
  const int column = (int)(unit - i * slices) * kSlice + lane_id() * kPer, left = hidden - column;
  if (left <= 0) return;
  const int word = word_of(ids, i, words);
  float v[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (word >= 0) {
    load_columns<DT>((const E*)table + (int64_t)word * hidden + column, left, v);
#pragma unroll
    for (int t = 0; t < kPer; ++t) v[t] *= scale;
  }
  store_columns<DT>((E*)out + i * hidden + column, left, v);
}

// the runs that are cut, as they come: the piece that one begins in, its word, how many pieces it has a part in
struct EmbeddingRuns {
  int32_t count, none[3];
  int4 runs[1];
};

// ---- tokens in the order of their words ----
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kSortRange = 1024, kSortList = 1024;
static_assert(kSortRange == 1 << 10 && kSortThreads == kSortRange, "a word of the range: ten bits, and a thread");
constexpr int kSortEach = 4, kSortBlock = kSortEach * kWave, kSortAhead = 4;      // neighbouring tokens of a lane, tokens of a wave at a time, loads under way

// the words of kSortEach tokens from i on, ~0 for those that do not count: outside the table, past the end, padding
template <typename I>
__device__ __forceinline__ void load_words(const I* __restrict__ ids, int64_t i, int64_t end, uint32_t words, uint32_t padding, uint32_t (&w)[kSortEach]) {
  I id[kSortEach];
  if (i + kSortEach <= end) {
    typedef I vector __attribute__((ext_vector_type(kSortEach), aligned(sizeof(I))));
    const vector v = *(const vector*)(ids + i);
#pragma unroll
    for (int t = 0; t < kSortEach; ++t) id[t] = v[t];
  } else {
#pragma unroll
    for (int t = 0; t < kSortEach; ++t) id[t] = i + t < end ? ids[i + t] : (I)-1;
  }
#pragma unroll
  for (int t = 0; t < kSortEach; ++t) w[t] = (uint64_t)(int64_t)id[t] < words && (uint32_t)id[t] != padding ? (uint32_t)id[t] : ~0u;
}

// Workgroup w: words [first, first + range).  Wave v of it goes through the tokens [v S, (v + 1) S), S a multiple of kSortBlock.
// order: the places of the tokens that count, stably by word; sorted: their words; starts[v]: how many are of smaller words than v, v = 0 .. words.
// crossing: emptied for the launch behind.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const I* __restrict__ ids, int64_t tokens, int words, int range, uint32_t padding,
                                                                      int32_t* __restrict__ order, int32_t* __restrict__ sorted, int32_t* __restrict__ starts,
                                                                      EmbeddingRuns* __restrict__ crossing) {
  __shared__ int32_t count[kSortWaves][kSortRange];
  __shared__ uint32_t list[kSortWaves][kSortList];      // a wave's tokens of this workgroup's words, in order: place in the wave's share, word in the range
  __shared__ int32_t sums[kSortWaves], below_of[kSortWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int first = (int)blockIdx.x * range, mine = words - first < range ? words - first : range;
  if (blockIdx.x == 0 && threadIdx.x == 0) crossing->count = 0;
  for (int r = threadIdx.x; r < kSortWaves * kSortRange; r += kSortThreads) (&count[0][0])[r] = 0;
  __syncthreads();
  const int64_t share = (tokens + kSortWaves * kSortBlock - 1) / (kSortWaves * kSortBlock) * kSortBlock;
  const int64_t begin = wave * share, end = begin + share < tokens ? begin + share : tokens;
  const uint64_t lower = (1ull << lane) - 1;
  // calls take(place of the lane's first token in the share, words) for kSortBlock tokens at a time, in order
  auto walk = [&](auto&& take) {
    for (int64_t at = begin; at < end; at += kSortAhead * kSortBlock) {
      uint32_t w[kSortAhead][kSortEach];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) load_words(ids, at + u * kSortBlock + lane * kSortEach, end, (uint32_t)words, padding, w[u]);
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) take((int)(at - begin + u * kSortBlock) + lane * kSortEach, w[u]);
    }
  };
  // for each word among up to a wave's tokens, of which those in `todo` count: each(word, the lanes that have it)
  auto match = [&](uint32_t word, uint64_t todo, auto&& each) {
    while (todo) {
      const uint32_t it = (uint32_t)__builtin_amdgcn_readlane((int)word, __builtin_ctzll(todo));
      const uint64_t same = __ballot(word == it) & todo;
      each((int)it, same);
      todo &= ~same;
    }
  };
  // the next places of word r for `n` tokens of the wave
  auto claim = [&](int r, int n) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&count[wave][r], n);
    return __builtin_amdgcn_readfirstlane(at);
  };
  int below = 0, listed = 0;
  walk([&](int place, const uint32_t (&w)[kSortEach]) {
    uint64_t here[kSortEach];
    int n = 0;
#pragma unroll
    for (int t = 0; t < kSortEach; ++t) {
      below += __popcll(__ballot(w[t] < (uint32_t)first));
      here[t] = __ballot(w[t] - (uint32_t)first < (uint32_t)mine);
      n += __popcll(here[t]);
    }
    if (n == 0) return;
    int to = listed;      // behind the tokens of the lanes below
#pragma unroll
    for (int t = 0; t < kSortEach; ++t) to += __popcll(here[t] & lower);
#pragma unroll
    for (int t = 0; t < kSortEach; ++t)
      if (here[t] >> lane & 1) {
        if (to < kSortList) list[wave][to] = (uint32_t)(place + t) << 10 | (w[t] - (uint32_t)first);
        ++to;
      }
    listed += n;
  });
  // more tokens than the list holds, as of a word that is much of the text: the share is gone through again instead, 64 tokens at a time
  const bool all_listed = listed <= kSortList && share <= 1 << 22;
  auto walk_all = [&](auto&& take) {
    for (int64_t at = begin; at < end; at += kWave) {
      const int64_t i = at + lane;
      const int64_t id = i < end ? (int64_t)ids[i] : -1;
      const uint32_t word = (uint64_t)id < (uint32_t)words && (uint32_t)id != padding ? (uint32_t)id - (uint32_t)first : ~0u;
      match(word, __ballot(word < (uint32_t)mine), [&](int r, uint64_t same) { take((int)i, r, same); });
    }
  };
  if (all_listed) {
    for (int i = lane; i < listed; i += kWave) atomicAdd(&count[wave][list[wave][i] & (kSortRange - 1)], 1);
  } else {
    walk_all([&](int, int r, uint64_t same) {
      if (lane == 0) atomicAdd(&count[wave][r], __popcll(same));
    });
  }
  if (lane == 0) below_of[wave] = below;
  __syncthreads();
  // thread r: word first + r
  const int r = threadIdx.x;
  int total = 0;
#pragma unroll
  for (int v = 0; v < kSortWaves; ++v) total += count[v][r];
  const int through = wave_inclusive_scan(total);
  if (lane == kWave - 1) sums[wave] = through;
  __syncthreads();
  int start = through - total;
#pragma unroll
  for (int v = 0; v < kSortWaves; ++v) start += below_of[v] + (v < wave ? sums[v] : 0);
  if (r < mine) {
    starts[first + r] = start;
    if (first + r == words - 1) starts[words] = start + total;
  }
#pragma unroll
  for (int v = 0; v < kSortWaves; ++v) {
    const int n = count[v][r];
    count[v][r] = start;
    start += n;
  }
  __syncthreads();
  auto put = [&](int place, int r, uint64_t same) {
    const int at = claim(r, __popcll(same));
    if (same >> lane & 1) {
      const int to = at + __popcll(same & lower);
      order[to] = place;
      sorted[to] = first + r;
    }
  };
  if (all_listed) {
    for (int i0 = 0; i0 < listed; i0 += kWave) {
      const uint32_t it = i0 + lane < listed ? list[wave][i0 + lane] : 0u;
      match(it & (kSortRange - 1), __ballot(i0 + lane < listed), [&](int r, uint64_t same) { put((int)begin + (int)(it >> 10), r, same); });
    }
  } else {
    walk_all(put);
  }
}

// ---- sums along the order ----
// Workgroups [0, piece_blocks): a wave per piece of kPiece places of the order and slice of columns; the others: rows of words without a token, zeroed.
// heads[p] / tails[p]: what the run that piece p begins inside of / ends inside of leaves there; a run that goes through the whole piece: heads[p].
// Words of a wave that zeroes (us a pass by 16 / 8 / 4 / 2 / 1: 32767 tokens, 100000 words of 2040 179 / 176 / 173 / 172 / 172; 2000 tokens, 128000 of 4096 225 / 222 / 219 / 218 / 220).
constexpr int kZeroRows = 2;
// A run of up to kWholeRun tokens is added up by the piece that it begins in, which has it in its lanes; longer ones are cut at the pieces' ends.
constexpr int kPiece = 32, kWholeRun = kWave - kPiece;

template <int DT>
__global__ void __launch_bounds__(kEmbThreads) embedding_sum_kernel(const void* __restrict__ grad, const int32_t* __restrict__ order, const int32_t* __restrict__ sorted,
                                                                    const int32_t* __restrict__ starts, int words, int hidden, int slices, int64_t piece_blocks,
                                                                    float scale, Sum<DT>* __restrict__ heads, Sum<DT>* __restrict__ tails, EmbeddingRuns* __restrict__ crossing,
                                                                    void* __restrict__ out, int64_t first_block) {
  typedef typename Elem<DT>::type E;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int64_t block = first_block + blockIdx.x;
  if (block >= piece_blocks) {
    const int64_t first = ((block - piece_blocks) * kEmbWaves + wave) * kZeroRows;
    if (first >= words) return;
    const int64_t v = first + lane;
    uint64_t todo = __ballot(lane < kZeroRows && v < words && starts[v < words ? v : words] == starts[v < words ? v + 1 : words]);
    const float none[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    while (todo) {
      E* const row = (E*)out + (first + __builtin_ctzll(todo)) * hidden;
      todo &= todo - 1;
      for (int column = lane * kPer; column < hidden; column += kSlice) store_columns<DT>(row + column, hidden - column, none);
    }
    return;
  }
  const int64_t unit = block * kEmbWaves + wave;
  const int64_t p = unit / slices, from = p * kPiece;
  const int total = starts[words];
  if (from >= total) return;
  const int column = (int)(unit - p * slices) * kSlice + lane * kPer, left = hidden - column;
  const int there = total - from < kWave ? (int)(total - from) : kWave, inside = there < kPiece ? there : kPiece;
  const int my_word = lane < there ? sorted[from + lane] : -1, my_place = lane < there ? order[from + lane] : 0;
  int word = __builtin_amdgcn_readlane(my_word, 0);
  const int last_word = __builtin_amdgcn_readlane(my_word, inside - 1);
  const int begin = starts[word], stop = starts[word + 1], last_begin = starts[last_word], last_stop = starts[last_word + 1];
  const bool from_others = begin < from && stop - begin <= kWholeRun;
  const int i0 = from_others ? (int)(stop - from) : 0;
  if (i0 >= inside) return;
  const int n = last_stop > from + inside && last_stop - last_begin <= kWholeRun ? (int)(last_stop - from) : inside;      // last_begin >= from: else i0 is past it
  const bool goes_on = last_stop > from + n;
  bool from_before = begin < from && !from_others;
  word = __builtin_amdgcn_readlane(my_word, i0);
  if (unit == p * slices && lane == 0 && goes_on && last_begin >= from)
    crossing->runs[atomicAdd(&crossing->count, 1)] = make_int4((int)p, last_word, (int)((last_stop - 1) / kPiece - p + 1), 0);
  // whole: all kPer columns are the row's
  auto add_up = [&](auto whole) {
    Sum<DT> acc[kPer] = {};
    auto keep = [&](Sum<DT>* parts) {
      Sum<DT>* const at = parts + p * hidden + column;
      if constexpr (decltype(whole)::value) {
        Sums<kPer, Sum<DT>> v;
#pragma unroll
        for (int t = 0; t < kPer; ++t) v.part[t / v.kEach][t % v.kEach] = acc[t];
        v.store(at);
      } else {
#pragma unroll
        for (int t = 0; t < kPer; ++t)
          if (t < left) at[t] = acc[t];
      }
    };
    auto finish = [&]() {     // the run of `word` ends here
      if (from_before) {
        keep(heads);
      } else {
        float v[kPer];
#pragma unroll
        for (int t = 0; t < kPer; ++t) v[t] = (float)(acc[t] * scale);
        store_columns<DT>((E*)out + (int64_t)word * hidden + column, left, v);
      }
    };
    constexpr int kAhead = 8;
    for (int i = i0; i < n; i += kAhead) {
      Piece<DT> v[kAhead];      // all under way before the first is looked at
      if constexpr (decltype(whole)::value) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          v[u].load((const E*)grad + (int64_t)__builtin_amdgcn_readlane(my_place, i + u < n ? i + u : n - 1) * hidden + column);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i + u < n) {
          const int here = __builtin_amdgcn_readlane(my_word, i + u);
          if (here != word) {
            finish();
            word = here;
            from_before = false;
#pragma unroll
            for (int t = 0; t < kPer; ++t) acc[t] = 0;
          }
          if constexpr (decltype(whole)::value) {
#pragma unroll
            for (int t = 0; t < kPer; ++t) acc[t] += v[u].value(t);
          } else {
            float last[kPer];
            load_columns<DT>((const E*)grad + (int64_t)__builtin_amdgcn_readlane(my_place, i + u) * hidden + column, left, last);
#pragma unroll
            for (int t = 0; t < kPer; ++t) acc[t] += last[t];
          }
        }
      }
    }
    if (!goes_on) finish();
    else keep(from_before ? heads : tails);
  };
  if (left >= kPer) add_up(std::true_type{});
  else if (left > 0) add_up(std::false_type{});
}

// ---- runs that are cut: a workgroup per run and kJoinColumns columns ----
constexpr int kJoinColumns = kWave * 4, kJoinThreads = 512, kJoinWaves = kJoinThreads / kWave, kJoinRuns = 128;

template <int DT>
__global__ void __launch_bounds__(kJoinThreads) embedding_join_kernel(int hidden, float scale, const Sum<DT>* __restrict__ heads, const Sum<DT>* __restrict__ tails,
                                                                      const EmbeddingRuns* __restrict__ crossing, void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  __shared__ Sum<DT> sums[kJoinWaves][kJoinColumns];
  const int wave = threadIdx.x / kWave, lane = lane_id(), column = (int)blockIdx.y * kJoinColumns + lane * 4;
  int4 it = crossing->runs[blockIdx.x];      // under way with the count: it may be none
  const int runs = crossing->count;
  for (int run = blockIdx.x; run < runs; run += gridDim.x) {
    if (run != (int)blockIdx.x) it = crossing->runs[run];
    const int64_t p = it.x, parts = it.z;
    const int word = it.y;
    // the waves take consecutive runs of the pieces' parts, and are added in order
    const int64_t share = (parts + kJoinWaves - 1) / kJoinWaves;
    const int64_t a = wave * share, b = a + share < parts ? a + share : parts;
    Sum<DT> acc[4] = {};
    auto row = [&](int64_t n) { return (n == 0 ? tails + p * hidden : heads + (p + n) * hidden) + column; };
    if (column + 4 <= hidden) {
      constexpr int kAhead = 8;
      for (int64_t i = a; i < b; i += kAhead) {
        Sums<4, Sum<DT>> v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u].load(row(i + u < b ? i + u : b - 1));
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i + u < b)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] += v[u].value(t);
      }
    } else {
      for (int64_t i = a; i < b; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (column + t < hidden) acc[t] += row(i)[t];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) sums[wave][lane * 4 + t] = acc[t];
    __syncthreads();
    const int c = (int)blockIdx.y * kJoinColumns + (int)threadIdx.x;
    if (threadIdx.x < kJoinColumns && c < hidden) {
      Sum<DT> v = 0;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) v += sums[w][threadIdx.x];
      ((E*)out)[(int64_t)word * hidden + c] = Elem<DT>::from_f32((float)(v * scale));
    }
    __syncthreads();      // the next run's sums
  }
}

// ---- up to kFewTokens tokens: the gradient by one launch ----
// A workgroup has up to kFewWords words and kFewSlices slices of the columns: it lists the tokens of those words, in order, and a wave adds up those of a word for a slice.
// Bound by the launch, or by the zeros of a large table.  Tokens of one word are added up one after the other, so it is for few of them (us of three launches / of this, forward
// included: 64 tokens, 1000 words of 64 19.2 / 5.9; 256 tokens, 128000 words of 2040 121 / 110; but 128 tokens of one word of 4096 17.2 / 19.0, 256 of them 18.2 / 35.5).
constexpr int kFewTokens = kEmbThreads, kFewWords = 16, kFewSlices = kEmbWaves;

template <int DT, typename I>
__global__ void __launch_bounds__(kEmbThreads) embedding_few_kernel(const void* __restrict__ grad, const I* __restrict__ ids, int tokens, int words, int each, int hidden,
                                                                    int slices, int padding, float scale, void* __restrict__ out, int64_t first_block) {
  typedef typename Elem<DT>::type E;
  __shared__ int32_t token_of[kFewTokens], place_of[kFewTokens], counts[kEmbWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int64_t first = (first_block + blockIdx.x) * each;
  int place = -1;
  if ((int)threadIdx.x < tokens) {
    const int word = word_of(ids, threadIdx.x, words);
    if (word >= first && word < first + each && word != padding) place = word - (int)first;
  }
  const uint64_t here = __ballot(place >= 0);
  if (lane == 0) counts[wave] = __popcll(here);
  __syncthreads();
  int to = __popcll(here & ((1ull << lane) - 1)), n = 0;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) {
    to += w < wave ? counts[w] : 0;
    n += counts[w];
  }
  if (place >= 0) {
    token_of[to] = threadIdx.x;
    place_of[to] = place;
  }
  __syncthreads();
  const int first_slice = (int)blockIdx.y * kFewSlices, my_slices = slices - first_slice < kFewSlices ? slices - first_slice : kFewSlices;
  const int units = (int)(words - first < each ? words - first : each) * my_slices;
  for (int unit = wave; unit < units; unit += kEmbWaves) {
    const int word = unit / my_slices, slice = first_slice + unit - word * my_slices, column = slice * kSlice + lane * kPer, left = hidden - column;
    const bool whole = hidden % kPer == 0 || (slice + 1) * kSlice <= hidden;      // every lane has eight columns or none
    Sum<DT> acc[kPer] = {};
    bool any = false;
    for (int c = 0; c < n; c += kWave) {
      const int token = c + lane < n ? token_of[c + lane] : 0;
      uint64_t todo = __ballot(c + lane < n && place_of[c + lane] == word);
      any = any || todo != 0;
      constexpr int kAhead = DT == MBX_F32 ? 8 : 16;
      while (todo) {
        const uint64_t now = todo;
        const int count = __popcll(now) < kAhead ? __popcll(now) : kAhead;
        int row[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          row[u] = __builtin_amdgcn_readlane(token, __builtin_ctzll(todo ? todo : now));
          todo &= todo - 1;      // 0 stays 0
        }
        if (whole) {
          Piece<DT> v[kAhead];      // all under way before the first is looked at
#pragma unroll
          for (int u = 0; u < kAhead; ++u) v[u].load((const E*)grad + (int64_t)row[u] * hidden + (left > 0 ? column : 0));
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (u < count)
#pragma unroll
              for (int t = 0; t < kPer; ++t) acc[t] += v[u].value(t);
        } else if (left > 0) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
            if (u < count) {
              float v[kPer];
              load_columns<DT>((const E*)grad + (int64_t)row[u] * hidden + column, left, v);
#pragma unroll
              for (int t = 0; t < kPer; ++t) acc[t] += v[t];
            }
        }
      }
    }
    float sums[kPer];
#pragma unroll
    for (int t = 0; t < kPer; ++t) sums[t] = any ? (float)(acc[t] * scale) : 0.f;
    if (left > 0) store_columns<DT>((E*)out + (first + word) * hidden + column, left, sums);
  }
}

struct EmbeddingParts {
  size_t order = 0, sorted = 0, starts = 0, heads = 0, tails = 0, crossing = 0, total = 0;
  int64_t pieces;
  EmbeddingParts(int64_t tokens, int words, int hidden) {
    pieces = ceil_div(tokens, kPiece);
    if (tokens <= kFewTokens) return;      // none
    auto take = [&](size_t bytes) {
      const size_t at = total;
      total += (bytes + 255) & ~(size_t)255;
      return at;
    };
    order = take((size_t)tokens * 4);
    sorted = take((size_t)tokens * 4);
    starts = take((size_t)(words + 1) * 4);
    heads = take((size_t)pieces * hidden * sizeof(Sum<MBX_F32>));      // enough for all types
    tails = take((size_t)pieces * hidden * sizeof(Sum<MBX_F32>));
    crossing = take(sizeof(EmbeddingRuns) + sizeof(int4) * (size_t)(pieces > kJoinRuns ? pieces : kJoinRuns));
  }
};

// launch(workgroups, the first of them) for all of them, in as many launches as that takes
template <typename F>
void in_launches(int64_t blocks, F&& launch) {
  for (int64_t first = 0; first < blocks; first += kEmbMaxBlocks) launch((unsigned)(blocks - first < kEmbMaxBlocks ? blocks - first : kEmbMaxBlocks), first);
}

template <int DT, typename I>
int launch_embedding(const void* ids, int64_t tokens, const void* table, int words, int hidden, float scale, void* out, hipStream_t s) {
  const int slices = (int)ceil_div(hidden, kSlice);
  in_launches(ceil_div(tokens * slices, kEmbWaves), [&](unsigned blocks, int64_t first) {
    embedding_kernel<DT, I><<<blocks, kEmbThreads, 0, s>>>((const I*)ids, tokens, table, words, hidden, slices, scale, out, first);
  });
  return launch_status();
}

template <typename I>
int launch_sort(const void* ids, int64_t tokens, int words, int64_t padding, int32_t* order, int32_t* sorted, int32_t* starts, EmbeddingRuns* crossing, hipStream_t s) {
  // a workgroup on every compute unit where there are words for them, and no more words each than it counts
  int range = (int)ceil_div(words, 256);
  if (range > kSortRange) range = kSortRange;
  embedding_sort_kernel<I><<<(unsigned)ceil_div(words, range), kSortThreads, 0, s>>>((const I*)ids, tokens, words, range, padding < 0 || padding >= words ? ~0u : (uint32_t)padding,
                                                                                     order, sorted, starts, crossing);
  return launch_status();
}

template <int DT>
int launch_sums(const void* grad, int words, int hidden, float scale, const EmbeddingParts& parts, char* scratch, void* out, hipStream_t s) {
  const int32_t *const order = (const int32_t*)(scratch + parts.order), *const sorted = (const int32_t*)(scratch + parts.sorted);
  const int32_t* const starts = (const int32_t*)(scratch + parts.starts);
  Sum<DT> *const heads = (Sum<DT>*)(scratch + parts.heads), *const tails = (Sum<DT>*)(scratch + parts.tails);
  EmbeddingRuns* const crossing = (EmbeddingRuns*)(scratch + parts.crossing);
  const int slices = (int)ceil_div(hidden, kSlice);
  const int64_t piece_blocks = ceil_div(parts.pieces * slices, kEmbWaves), zero_blocks = ceil_div(words, kEmbWaves * kZeroRows);
  in_launches(piece_blocks + zero_blocks, [&](unsigned blocks, int64_t first) {
    embedding_sum_kernel<DT><<<blocks, kEmbThreads, 0, s>>>(grad, order, sorted, starts, words, hidden, slices, piece_blocks, scale, heads, tails, crossing, out, first);
  });
  if (const int rc = launch_status()) return rc;
  if (parts.pieces > 1) {
    const unsigned runs = (unsigned)(parts.pieces - 1 < kJoinRuns ? parts.pieces - 1 : kJoinRuns);
    embedding_join_kernel<DT><<<dim3(runs, (unsigned)ceil_div(hidden, kJoinColumns)), kJoinThreads, 0, s>>>(hidden, scale, heads, tails, crossing, out);
    return launch_status();
  }
  return 0;
}

template <int DT, typename I>
int launch_few(const void* grad, const void* ids, int tokens, int words, int hidden, int64_t padding, float scale, void* out, hipStream_t s) {
  const int slices = (int)ceil_div(hidden, kSlice), each = words <= 256 ? 1 : words >= 256 * kFewWords ? kFewWords : (int)ceil_div(words, 256);
  in_launches(ceil_div(words, each), [&](unsigned blocks, int64_t first) {
    embedding_few_kernel<DT, I><<<dim3(blocks, (unsigned)ceil_div(slices, kFewSlices)), kEmbThreads, 0, s>>>(
        grad, (const I*)ids, tokens, words, each, hidden, slices, padding < 0 || padding >= words ? -1 : (int)padding, scale, out, first);
  });
  return launch_status();
}

bool embedding_sizes_ok(int64_t tokens, int64_t words, int64_t hidden) { return tokens >= 0 && words >= 0 && hidden >= 0; }
// 32-bit places of tokens; the join's grid counts columns in 16 bits
bool embedding_in_range(int64_t tokens, int64_t words, int64_t hidden) {
  return tokens <= 0x7fffff00 && words <= 0x7ffffffe && hidden <= (int64_t)65535 * kJoinColumns;
}

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

int mbx_embedding(const void* ids, int itype, int64_t tokens, const void* table, int dtype, int64_t words, int64_t hidden, float scale, void* out, mbx_stream_t stream) {
  if (!embedding_sizes_ok(tokens, words, hidden) || (itype != MBX_I32 && itype != MBX_I64) || dtype < MBX_BF16 || dtype > MBX_F32 || !std::isfinite(scale)) return MBX_EINVAL;
  if (!embedding_in_range(tokens, words, hidden)) return MBX_ERANGE;
  if (tokens == 0 || hidden == 0) return 0;
  if (!ids || !out || (words > 0 && !table)) return MBX_EINVAL;
  hipStream_t s = as_stream(stream);
#define MBX_EMBEDDING(DT) (itype == MBX_I32 ? launch_embedding<DT, int32_t>(ids, tokens, table, (int)words, (int)hidden, scale, out, s) \
                                            : launch_embedding<DT, int64_t>(ids, tokens, table, (int)words, (int)hidden, scale, out, s))
  return dtype == MBX_BF16 ? MBX_EMBEDDING(MBX_BF16) : dtype == MBX_F16 ? MBX_EMBEDDING(MBX_F16) : MBX_EMBEDDING(MBX_F32);
#undef MBX_EMBEDDING
}

size_t mbx_embedding_gradient_scratch_bytes(int64_t tokens, int64_t words, int64_t hidden) {
  if (!embedding_sizes_ok(tokens, words, hidden) || !embedding_in_range(tokens, words, hidden)) return 0;
  return EmbeddingParts(tokens, (int)words, (int)hidden).total;
}

int mbx_embedding_gradient(const void* grad, const void* ids, int itype, int64_t tokens, int dtype, int64_t words, int64_t hidden, int64_t padding, float scale,
                           void* out, void* scratch, size_t scratch_bytes, mbx_stream_t stream) {
  if (!embedding_sizes_ok(tokens, words, hidden) || (itype != MBX_I32 && itype != MBX_I64) || dtype < MBX_BF16 || dtype > MBX_F32 || !std::isfinite(scale)) return MBX_EINVAL;
  if (!embedding_in_range(tokens, words, hidden)) return MBX_ERANGE;
  if (words == 0 || hidden == 0) return 0;
  if (!out || (tokens > 0 && (!ids || !grad))) return MBX_EINVAL;
  if (tokens <= kFewTokens) {
#define MBX_FEW(DT) (itype == MBX_I32 ? launch_few<DT, int32_t>(grad, ids, (int)tokens, (int)words, (int)hidden, padding, scale, out, as_stream(stream)) \
                                      : launch_few<DT, int64_t>(grad, ids, (int)tokens, (int)words, (int)hidden, padding, scale, out, as_stream(stream)))
    return dtype == MBX_BF16 ? MBX_FEW(MBX_BF16) : dtype == MBX_F16 ? MBX_FEW(MBX_F16) : MBX_FEW(MBX_F32);
#undef MBX_FEW
  }
  const EmbeddingParts parts(tokens, (int)words, (int)hidden);
  if (!scratch || scratch_bytes < parts.total || ((uintptr_t)scratch & 15)) return MBX_ESCRATCH;
  char* const base = (char*)scratch;
  hipStream_t s = as_stream(stream);
  int32_t *const order = (int32_t*)(base + parts.order), *const sorted = (int32_t*)(base + parts.sorted), *const starts = (int32_t*)(base + parts.starts);
  EmbeddingRuns* const crossing = (EmbeddingRuns*)(base + parts.crossing);
  const int rc = itype == MBX_I32 ? launch_sort<int32_t>(ids, tokens, (int)words, padding, order, sorted, starts, crossing, s)
                                  : launch_sort<int64_t>(ids, tokens, (int)words, padding, order, sorted, starts, crossing, s);
  if (rc) return rc;
  if (dtype == MBX_BF16) return launch_sums<MBX_BF16>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
  if (dtype == MBX_F16) return launch_sums<MBX_F16>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
  return launch_sums<MBX_F32>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
}

}  // extern "C"
