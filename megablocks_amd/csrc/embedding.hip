// Rows of a table by token, times a scale, and the gradient of the table.
//
//   out[i] = scale table[ids[i]]           dtable[v] = scale sum over {i : ids[i] = v} of dout[i], i ascending
//
// Both are bound by memory: the rows read and written once, for the gradient the whole table written, most of it zeros.  The gradient's sums are fp32 in
// a fixed order: rows are added along the tokens sorted by word (stably), kPiece of them by a wave, whose runs of one word that end inside go straight
// to the table; what a run that crosses pieces leaves in each is kept in fp32 and added up, in order, by a launch of its own.  So a word that is half of the text
// costs no more than any other, and results do not depend on timing: no atomics.
//
// Sorting: workgroup w owns a range of words and goes through all tokens twice, once to count its own and those of smaller words, once to place them: no
// exchange between workgroups, one launch.
//
// A token outside the table gives a row of zeros and no gradient.  Tensors may start anywhere and rows have any length: the memory unit takes 16-byte
// accesses at any address.
#include "common.h"

namespace mbx {
namespace {

typedef uint32_t u32x4e __attribute__((ext_vector_type(4)));
typedef u32x4e __attribute__((aligned(2))) u32x4_at2;
typedef u32x4e __attribute__((aligned(4))) u32x4_at4;

constexpr int kEmbThreads = 256, kEmbWaves = kEmbThreads / kWave;
constexpr int kPer = 8;                               // columns of a lane
constexpr int kSlice = kPer * kWave;                  // columns of a wave

template <int DT>
__device__ __forceinline__ void load8(const void* at, float (&v)[kPer]) {
  if constexpr (DT == MBX_F32) {
    const u32x4e a = *(const u32x4_at4*)at, b = *(const u32x4_at4*)((const float*)at + 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) { v[t] = __uint_as_float(a[t]); v[4 + t] = __uint_as_float(b[t]); }
  } else {
    const u32x4e a = *(const u32x4_at2*)at;
#pragma unroll
    for (int t = 0; t < kPer; ++t)
      v[t] = Elem<DT>::to_f32(__builtin_bit_cast(typename Elem<DT>::type, (uint16_t)(a[t >> 1] >> ((t & 1) * 16))));
  }
}

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

// up to kPer columns from `at`, of which `left` are the row's
template <int DT>
__device__ __forceinline__ void load_columns(const void* at, int left, float (&v)[kPer]) {
  if (left >= kPer) {
    load8<DT>(at, v);
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
                                                                int slices, float scale, void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  const int64_t unit = (int64_t)blockIdx.x * kEmbWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
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

// ---- tokens in the order of their words ----
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kSortRange = 1024, kSortAhead = 8;

// Workgroup w: words [first, first + range).  Wave v of it goes through the tokens [v S, (v + 1) S), S a multiple of 64.
// order: the places of the tokens that count, stably by word; sorted: their words; starts[v]: how many are of smaller words than v, v = 0 .. words.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const I* __restrict__ ids, int64_t tokens, int words, int range, int padding,
                                                                      int32_t* __restrict__ order, int32_t* __restrict__ sorted, int32_t* __restrict__ starts) {
  __shared__ int32_t count[kSortWaves][kSortRange];
  __shared__ int32_t sums[kSortWaves], below_of[kSortWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int first = (int)blockIdx.x * range, mine = words - first < range ? words - first : range;
  for (int r = threadIdx.x; r < kSortWaves * kSortRange; r += kSortThreads) (&count[0][0])[r] = 0;
  __syncthreads();
  const int64_t share = (tokens + kSortThreads - 1) / kSortThreads * kWave;
  const int64_t begin = wave * share, end = begin + share < tokens ? begin + share : tokens;
  // calls take(place, word or -1) for 64 tokens at a time
  auto walk = [&](auto&& take) {
    for (int64_t at = begin; at < end; at += kSortAhead * kWave) {
      int word[kSortAhead];
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) {
        const int64_t i = at + u * kWave + lane;
        word[u] = i < end ? word_of(ids, i, words) : -1;
        if (word[u] == padding) word[u] = -1;
      }
#pragma unroll
      for (int u = 0; u < kSortAhead; ++u) take((int)(at + u * kWave) + lane, word[u]);
    }
  };
  // for each word of this workgroup's among the wave's 64 tokens: each(its place in the range, the lanes that have it)
  auto match = [&](int word, auto&& each) {
    uint64_t todo = __ballot((unsigned)(word - first) < (unsigned)mine && word >= 0);
    while (todo) {
      const int it = __builtin_amdgcn_readlane(word, __builtin_ctzll(todo));
      const uint64_t same = __ballot(word == it);
      each(it - first, same);
      todo &= ~same;
    }
  };
  int below = 0;
  walk([&](int, int word) {
    below += word >= 0 && word < first ? 1 : 0;
    match(word, [&](int r, uint64_t same) {
      if (lane == 0) count[wave][r] += __popcll(same);
    });
  });
#pragma unroll
  for (int off = 32; off; off >>= 1) below += __shfl_xor(below, off, kWave);
  if (lane == 0) below_of[wave] = below;
  __syncthreads();
  // thread r: word first + r
  const int r = threadIdx.x;
  int total = 0;
  for (int v = 0; v < kSortWaves; ++v) total += count[v][r];
  const int through = wave_inclusive_scan(total);
  if (lane == kWave - 1) sums[wave] = through;
  __syncthreads();
  int start = through - total;
  for (int v = 0; v < kSortWaves; ++v) start += below_of[v] + (v < wave ? sums[v] : 0);
  if (r < mine) {
    starts[first + r] = start;
    if (first + r == words - 1) starts[words] = start + total;
  }
  for (int v = 0; v < kSortWaves; ++v) {
    const int n = count[v][r];
    count[v][r] = start;
    start += n;
  }
  __syncthreads();
  walk([&](int place, int word) {
    match(word, [&](int r, uint64_t same) {
      const int at = count[wave][r];
      if (word == r + first) {
        const int to = at + __popcll(same & ((1ull << lane) - 1));
        order[to] = place;
        sorted[to] = word;
      }
      if (lane == 0) count[wave][r] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");     // the other lanes read it for the next word
    });
  });
}

// ---- sums along the order ----
// Workgroups [0, piece_blocks): a wave per piece of `piece` places of the order and slice of columns; the others: rows of words without a token, zeroed.
// heads[p] / tails[p]: what the run that piece p begins inside of / ends inside of leaves there; a run that goes through the whole piece: heads[p].
constexpr int kZeroRows = 64;    // words of a wave

template <int DT>
__global__ void __launch_bounds__(kEmbThreads) embedding_sum_kernel(const void* __restrict__ grad, const int32_t* __restrict__ order, const int32_t* __restrict__ sorted,
                                                                    const int32_t* __restrict__ starts, int words, int hidden, int slices, int piece, int64_t piece_blocks,
                                                                    float scale, float* __restrict__ heads, float* __restrict__ tails, void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  if ((int64_t)blockIdx.x >= piece_blocks) {
    const int64_t first = (((int64_t)blockIdx.x - piece_blocks) * kEmbWaves + wave) * kZeroRows;
    if (first >= words) return;
    const int64_t v = first + lane;
    uint64_t todo = __ballot(v < words && starts[v < words ? v : words] == starts[v < words ? v + 1 : words]);
    const float none[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    while (todo) {
      E* const row = (E*)out + (first + __builtin_ctzll(todo)) * hidden;
      todo &= todo - 1;
      for (int column = lane * kPer; column < hidden; column += kSlice) store_columns<DT>(row + column, hidden - column, none);
    }
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * kEmbWaves + wave;
  const int64_t p = unit / slices, from = p * piece;
  const int total = starts[words];
  if (from >= total) return;
  const int column = (int)(unit - p * slices) * kSlice + lane * kPer, left = hidden - column;
  const int n = total - from < piece ? (int)(total - from) : piece;          // up to a wave's lanes
  const int my_word = lane < n ? sorted[from + lane] : -1, my_place = lane < n ? order[from + lane] : 0;
  int word = __builtin_amdgcn_readlane(my_word, 0);
  bool from_before = from > 0 && sorted[from - 1] == word;
  float acc[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto keep = [&](float* parts) {
    if (left > 0) store_columns<MBX_F32>(parts + p * hidden + column, left, acc);
  };
  auto finish = [&]() {     // the run of `word` ends here
    if (from_before) {
      keep(heads);
    } else if (left > 0) {
      float v[kPer];
#pragma unroll
      for (int t = 0; t < kPer; ++t) v[t] = acc[t] * scale;
      store_columns<DT>((E*)out + (int64_t)word * hidden + column, left, v);
    }
  };
  constexpr int kAhead = 8;
  for (int i = 0; i < n; i += kAhead) {
    float v[kAhead][kPer];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i + u < n && left > 0)
        load_columns<DT>((const E*)grad + (int64_t)__builtin_amdgcn_readlane(my_place, i + u) * hidden + column, left, v[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u < n) {
        const int here = __builtin_amdgcn_readlane(my_word, i + u);
        if (here != word) {
          finish();
          word = here;
          from_before = false;
#pragma unroll
          for (int t = 0; t < kPer; ++t) acc[t] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < kPer; ++t) acc[t] += v[u][t];
      }
    }
  }
  const bool goes_on = from + n < total && sorted[from + n] == word;
  if (goes_on) keep(from_before ? heads : tails);
  else finish();
}

// ---- runs that cross pieces: a workgroup per piece that such a run begins in and kJoinColumns columns ----
constexpr int kJoinColumns = kWave * 4;

template <int DT>
__global__ void __launch_bounds__(kEmbThreads) embedding_join_kernel(const int32_t* __restrict__ sorted, const int32_t* __restrict__ starts, int words, int hidden,
                                                                     int piece, float scale, const float* __restrict__ heads, const float* __restrict__ tails,
                                                                     void* __restrict__ out) {
  typedef typename Elem<DT>::type E;
  __shared__ float sums[kEmbWaves][kJoinColumns];
  const int64_t p = blockIdx.x, from = p * piece;
  const int total = starts[words];
  if (from + piece >= total) return;                     // nothing behind this piece
  const int word = sorted[from + piece - 1];
  const int begin = starts[word], end = starts[word + 1];
  if (begin < from || end <= from + piece) return;
  const int64_t last = (end - 1) / piece;                // pieces p .. last
  const int wave = threadIdx.x / kWave, lane = lane_id(), column = (int)blockIdx.y * kJoinColumns + lane * 4;
  // the waves take consecutive runs of the pieces' parts, and are added in order
  const int64_t parts = last - p + 1, share = (parts + kEmbWaves - 1) / kEmbWaves;
  const int64_t a = wave * share, b = a + share < parts ? a + share : parts;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t i = a; i < b; ++i) {
    const float* const row = (i == 0 ? tails + p * hidden : heads + (p + i) * hidden) + column;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (column + t < hidden) acc[t] += row[t];
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) sums[wave][lane * 4 + t] = acc[t];
  __syncthreads();
  const int c = (int)blockIdx.y * kJoinColumns + (int)threadIdx.x;
  if (c >= hidden) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) v += sums[w][threadIdx.x];
  ((E*)out)[(int64_t)word * hidden + c] = Elem<DT>::from_f32(v * scale);
}
static_assert(kJoinColumns == kEmbThreads, "a column a thread");

struct EmbeddingParts {
  size_t order, sorted, starts, heads, tails, total = 0;
  int piece;
  int64_t pieces;
  EmbeddingParts(int64_t tokens, int words, int hidden) {
    piece = tokens <= (1 << 17) ? 32 : 64;
    pieces = ceil_div(tokens, piece);
    auto take = [&](size_t bytes) {
      const size_t at = total;
      total += (bytes + 255) & ~(size_t)255;
      return at;
    };
    order = take((size_t)tokens * 4);
    sorted = take((size_t)tokens * 4);
    starts = take((size_t)(words + 1) * 4);
    heads = take((size_t)pieces * hidden * 4);
    tails = take((size_t)pieces * hidden * 4);
  }
};

template <int DT, typename I>
int launch_embedding(const void* ids, int64_t tokens, const void* table, int words, int hidden, float scale, void* out, hipStream_t s) {
  const int slices = (int)ceil_div(hidden, kSlice);
  const int64_t blocks = ceil_div(tokens * slices, kEmbWaves);
  if (blocks > 0x7fffffff) return MBX_ERANGE;
  embedding_kernel<DT, I><<<(unsigned)blocks, kEmbThreads, 0, s>>>((const I*)ids, tokens, table, words, hidden, slices, scale, out);
  return launch_status();
}

template <typename I>
int launch_sort(const void* ids, int64_t tokens, int words, int64_t padding, int32_t* order, int32_t* sorted, int32_t* starts, hipStream_t s) {
  // a workgroup on every compute unit where there are words for them, and no more words each than it counts
  int range = (int)ceil_div(words, 256);
  if (range > kSortRange) range = kSortRange;
  embedding_sort_kernel<I><<<(unsigned)ceil_div(words, range), kSortThreads, 0, s>>>((const I*)ids, tokens, words, range, padding < 0 || padding >= words ? -2 : (int)padding,
                                                                                     order, sorted, starts);
  return launch_status();
}

template <int DT>
int launch_sums(const void* grad, int words, int hidden, float scale, const EmbeddingParts& parts, char* scratch, void* out, hipStream_t s) {
  const int32_t *const order = (const int32_t*)(scratch + parts.order), *const sorted = (const int32_t*)(scratch + parts.sorted);
  const int32_t* const starts = (const int32_t*)(scratch + parts.starts);
  float *const heads = (float*)(scratch + parts.heads), *const tails = (float*)(scratch + parts.tails);
  const int slices = (int)ceil_div(hidden, kSlice);
  const int64_t piece_blocks = ceil_div(parts.pieces * slices, kEmbWaves), zero_blocks = ceil_div(words, kEmbWaves * kZeroRows);
  if (piece_blocks + zero_blocks > 0x7fffffff) return MBX_ERANGE;
  embedding_sum_kernel<DT><<<(unsigned)(piece_blocks + zero_blocks), kEmbThreads, 0, s>>>(grad, order, sorted, starts, words, hidden, slices, parts.piece, piece_blocks,
                                                                                          scale, heads, tails, out);
  if (const int rc = launch_status()) return rc;
  if (parts.pieces > 1) {
    embedding_join_kernel<DT><<<dim3((unsigned)(parts.pieces - 1), (unsigned)ceil_div(hidden, kJoinColumns)), kEmbThreads, 0, s>>>(sorted, starts, words, hidden, parts.piece,
                                                                                                                              scale, heads, tails, out);
    return launch_status();
  }
  return 0;
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
  if (!embedding_sizes_ok(tokens, words, hidden) || (itype != MBX_I32 && itype != MBX_I64) || dtype < MBX_BF16 || dtype > MBX_F32) return MBX_EINVAL;
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
  if (!embedding_sizes_ok(tokens, words, hidden) || (itype != MBX_I32 && itype != MBX_I64) || dtype < MBX_BF16 || dtype > MBX_F32) return MBX_EINVAL;
  if (!embedding_in_range(tokens, words, hidden)) return MBX_ERANGE;
  if (words == 0 || hidden == 0) return 0;
  if (!out || (tokens > 0 && (!ids || !grad))) return MBX_EINVAL;
  const EmbeddingParts parts(tokens, (int)words, (int)hidden);
  if (!scratch || scratch_bytes < parts.total || ((uintptr_t)scratch & 15)) return MBX_ESCRATCH;
  char* const base = (char*)scratch;
  hipStream_t s = as_stream(stream);
  int32_t *const order = (int32_t*)(base + parts.order), *const sorted = (int32_t*)(base + parts.sorted), *const starts = (int32_t*)(base + parts.starts);
  const int rc = itype == MBX_I32 ? launch_sort<int32_t>(ids, tokens, (int)words, padding, order, sorted, starts, s)
                                  : launch_sort<int64_t>(ids, tokens, (int)words, padding, order, sorted, starts, s);
  if (rc) return rc;
  if (dtype == MBX_BF16) return launch_sums<MBX_BF16>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
  if (dtype == MBX_F16) return launch_sums<MBX_F16>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
  return launch_sums<MBX_F32>(grad, (int)words, (int)hidden, scale, parts, base, out, s);
}

}  // extern "C"
