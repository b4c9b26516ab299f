// The choice of experts by softmax or sigmoid scores, with a bias that keeps the experts in balance, by groups, its gradient, and the
// update of the bias.
//
//   s = softmax(x) or 1 / (1 + exp(-x));  key = s + bias, without a bias x itself, whose order is the same
//   group key = the sum of the group's `group_best` (1, 2) largest keys (without a bias: scores); the `top_groups` largest are open
//   indices = the top_k open experts of largest key, in descending order; ties go to the lower index, NaN comes first
//   weights = scale s[indices] / ||s[indices]||_p
//
// The order is that of the exact keys.  Scores in fp32 are off by some 2^-23, and of 256 scores of a token two neighbours in the order are closer
// than that once in a few thousand tokens: where two keys next to each other in the order are within kCloseKeys without being made of the same logit and
// bias, or the last chosen one and the largest left out that is not made of the same, the wave does the choice over with keys in 64 bits.
//
// LANES (16 or 64) lanes have a token, R experts in a row each, so that a lane reads and writes its experts as one piece and most groups are a
// power of two of neighbouring lanes.  What bounds it is instructions: a token's rounds of "largest of all, then its place" (top_k + 1 of them) take most.
// 32768 tokens, 8 of 256 experts in 8 groups with a bias, bf16: 32 us for 36 MB, its gradient 14.5 us for 53 MB (1.1 and 3.7 TB/s).
// Softmax scores of experts that are nearly alike take longer with a bias, since kCloseKeys goes by 1 and not by the scores: 8 of 256 experts, biases of zero, logits
// of deviation 1.5 / 0.1 / 0.02, bf16 21 / 21 / 67 us, fp32 31 / 55 / 78; 512 experts, fp32, 61 / 107 / 127.
#include "common.h"

namespace mbx {
namespace {

constexpr int kChooseThreads = 256;
constexpr int kChooseMaxExperts = 512, kChooseMaxTopK = 64, kChooseMaxGroups = 64;
constexpr float kCloseKeys = 0x1p-19f;   // of 1 + |key|: 16 times what the keys are off by

struct Choose {
  const void* logits;
  const float* bias;
  int64_t tokens;
  int experts, top_k, sigmoid, groups, top_groups, group_best;
  float norm_p, scale;
  void* scores;
  void* weights;
  int64_t* indices;
  int32_t* indices32;
  float* lse;
  int64_t first;   // the launch's first token
};

// ---- between the LANES lanes of a token ----

template <int CTRL, typename T>
__device__ __forceinline__ T dpp(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
  }
}

// v of the rows of 16 (half waves) and of the other row of the pair (half wave), as first(..) and second(..)
template <bool HALVES, typename T>
__device__ __forceinline__ void swapped(T v, T& first, T& second) {
  const auto swap = [](uint32_t x) {
    if constexpr (HALVES) return __builtin_amdgcn_permlane32_swap(x, x, false, false);
    else return __builtin_amdgcn_permlane16_swap(x, x, false, false);
  };
  if constexpr (sizeof(T) == 4) {
    const auto p = swap(__builtin_bit_cast(uint32_t, v));
    first = __builtin_bit_cast(T, (uint32_t)p[0]);
    second = __builtin_bit_cast(T, (uint32_t)p[1]);
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    first = __builtin_bit_cast(T, (uint64_t)(uint32_t)hi[0] << 32 | (uint32_t)lo[0]);
    second = __builtin_bit_cast(T, (uint64_t)(uint32_t)hi[1] << 32 | (uint32_t)lo[1]);
  }
}

constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// all lanes of a token get v combined over them, for a commutative op
template <int LANES, typename T, typename F>
__device__ __forceinline__ T over_token(T v, F&& op) {
  v = op(v, dpp<kQuadXor1>(v));
  v = op(v, dpp<kQuadXor2>(v));
  v = op(v, dpp<kHalfMirror>(v));   // the lanes of a quad are alike
  v = op(v, dpp<kMirror>(v));
  if constexpr (LANES == 64) {
    T a, b;
    swapped<false>(v, a, b);
    v = op(a, b);
    swapped<true>(v, a, b);
    v = op(a, b);
  }
  return v;
}

template <typename T> __device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
template <typename T> __host__ __device__ __forceinline__ T smaller(T a, T b) { return a < b ? a : b; }

template <int LANES, typename T> __device__ __forceinline__ T token_max(T v) { return over_token<LANES>(v, [](T a, T b) { return larger(a, b); }); }
template <int LANES, typename T> __device__ __forceinline__ T token_min(T v) { return over_token<LANES>(v, [](T a, T b) { return smaller(a, b); }); }
template <int LANES, typename T> __device__ __forceinline__ T token_sum(T v) { return over_token<LANES>(v, [](T a, T b) { return a + b; }); }

// ---- keys as whole numbers in their order: 0 stands for "not a candidate", the largest for NaN ----

__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);   // -0 as 0
  return v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.);
  return v != v ? ~0ull : (u >> 63) ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ float unordered(uint32_t u) { return u == 0xffffffffu ? NAN : __builtin_bit_cast(float, (u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ double unordered(uint64_t u) {
  return u == ~0ull ? (double)NAN : __builtin_bit_cast(double, (u >> 63) ? u & ~(1ull << 63) : ~u);
}

template <typename F> struct Keys;
template <> struct Keys<float> { typedef uint32_t type; };
template <> struct Keys<double> { typedef uint64_t type; };

// The open groups of a token as a bit each, given its experts' keys (0: none).  close: whether two groups on either side of the border are
// within what the keys may be off by, which goes by the sizes of the keys that are added up: large biases may leave little of them.
template <int LANES, int R, typename F>
__device__ __forceinline__ uint64_t open_groups(const typename Keys<F>::type (&key)[R], const Choose& c, int lane, bool& close) {
  typedef typename Keys<F>::type U;
  const int size = c.experts / c.groups, base = lane * R;
  const auto merge = [](U& m1, U& m2, U a1, U a2) {
    const U low = smaller(m1, a1);
    m1 = larger(m1, a1);
    m2 = larger(low, larger(m2, a2));   // at most one of m2 and a2 is above `low`
  };
  const auto value = [&](U m1, U m2) {
    const F first = unordered(m1);
    return c.group_best == 2 && m2 != 0 ? first + unordered(m2) : first;
  };
  const auto off_by = [&](U m1, U m2) {
    const F first = unordered(m1), second = c.group_best == 2 && m2 != 0 ? unordered(m2) : (F)0;
    return (F)kCloseKeys * (1 + (first < 0 ? -first : first) + (second < 0 ? -second : second));
  };
  F mine = 0, off = 0;   // of group `lane`
  const int per = size / R;
  if (per * R == size && per > 0 && (per & (per - 1)) == 0) {   // a group is `per` lanes next to each other
    U m1 = 0, m2 = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) merge(m1, m2, key[r], 0);
    if (per > 1) merge(m1, m2, dpp<kQuadXor1>(m1), dpp<kQuadXor1>(m2));
    if (per > 2) merge(m1, m2, dpp<kQuadXor2>(m1), dpp<kQuadXor2>(m2));
    if (per > 4) merge(m1, m2, dpp<kHalfMirror>(m1), dpp<kHalfMirror>(m2));
    if (per > 8) merge(m1, m2, dpp<kMirror>(m1), dpp<kMirror>(m2));
    if constexpr (LANES == 64) {
      U a1, a2;
      if (per > 16) { swapped<false>(m1, m1, a1); swapped<false>(m2, m2, a2); merge(m1, m2, a1, a2); }
      if (per > 32) { swapped<true>(m1, m1, a1); swapped<true>(m2, m2, a2); merge(m1, m2, a1, a2); }
    }
    const int from = lane * per < LANES ? lane * per : 0;
    mine = __shfl(value(m1, m2), from, LANES);
    off = __shfl(off_by(m1, m2), from, LANES);
  } else {
#pragma unroll 1
    for (int g = 0; g < c.groups; ++g) {
      U m1 = 0, m2 = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int e = base + r;
        merge(m1, m2, e >= g * size && e < (g + 1) * size ? key[r] : 0, 0);
      }
      merge(m1, m2, dpp<kQuadXor1>(m1), dpp<kQuadXor1>(m2));
      merge(m1, m2, dpp<kQuadXor2>(m1), dpp<kQuadXor2>(m2));
      merge(m1, m2, dpp<kHalfMirror>(m1), dpp<kHalfMirror>(m2));
      merge(m1, m2, dpp<kMirror>(m1), dpp<kMirror>(m2));
      if constexpr (LANES == 64) {
        U a1, a2;
        swapped<false>(m1, m1, a1); swapped<false>(m2, m2, a2); merge(m1, m2, a1, a2);
        swapped<true>(m1, m1, a1); swapped<true>(m2, m2, a2); merge(m1, m2, a1, a2);
      }
      if (lane == g) {
        mine = value(m1, m2);
        off = off_by(m1, m2);
      }
    }
  }
  const U order = ordered(mine);
  int before = 0;
#pragma unroll 1
  for (int g = 0; g < c.groups; ++g) {
    const U other = __shfl(order, g, LANES);
    before += other > order || (other == order && g < lane) ? 1 : 0;
  }
  const bool group = lane < c.groups, open = group && before < c.top_groups;
  const F lowest = token_min<LANES>(open ? mine - off : (F)INFINITY), highest = token_max<LANES>(group && !open ? mine + off : (F)-INFINITY);
  close = !(lowest > highest) || (group && !(off < (F)INFINITY));
  const uint64_t all = __ballot(open);
  return LANES == 64 ? all : (all >> (lane_id() & ~(LANES - 1))) & 0xffffu;
}

// Keys of experts of closed groups, and of lanes' places past the last expert, as 0.
template <int R, typename U>
__device__ __forceinline__ void keep_open(U (&key)[R], uint64_t open, int base, int size) {
  if (size % R == 0) {   // a lane is in one group
    const bool in = (open >> (base / size)) & 1;
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = in ? key[r] : 0;
    return;
  }
  int g = base / size, in = base - g * size;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    key[r] = (open >> g) & 1 ? key[r] : 0;
    const bool next = ++in == size;
    in = next ? 0 : in;
    g += next ? 1 : 0;
  }
}
template <int R, bool WHOLE, typename U, typename F>
__device__ __forceinline__ void order_keys(U (&key)[R], const F (&v)[R], int base, int experts) {
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = base + (WHOLE ? 0 : r) < experts ? ordered(v[r]) : 0;
}

// The experts of the `count` largest keys, in order: lane j has the j-th in `mine`; the one after the first top_k in `next`.
template <int LANES, int R, typename U>
__device__ __forceinline__ void pick(U (&key)[R], int lane, int top_k, int count, int& mine, int& next) {
  const int base = lane * R;
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    U best = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) best = larger(best, key[r]);
    best = token_max<LANES>(best);
    int place = R;     // places of the lane, not experts: numbers that the instructions hold
#pragma unroll
    for (int r = R - 1; r >= 0; --r) place = key[r] == best ? r : place;
    const int e = token_min<LANES>(place == R ? 0x7fffffff : base + place);
    if (j == top_k) next = e;
    else if (lane == j) mine = e;
    place = e - base;
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = place == r ? 0 : key[r];
  }
}

// Where 16-bit numbers come out, the quick exponential and reciprocal do: they are off by a few 2^-24 of the largest score.  So they do for lse, which is fp32 of
// 16-bit logits: the sum of the exponentials is off by as much of itself, the logits by 2^-9 or 2^-12 of themselves.
template <int DT> __device__ __forceinline__ float exp_of(float v) { return DT == MBX_F32 ? expf(v) : __expf(v); }
template <int DT> __device__ __forceinline__ float over(float a, float b) { return DT == MBX_F32 ? a / b : a * __builtin_amdgcn_rcpf(b); }

// ||w||_p of w >= 0 over a token's lanes, as the largest times the norm of w over that: sigmoid scores of 1e-20, or large p, have powers below fp32
template <int LANES>
__device__ __forceinline__ float token_pnorm(float w, float p) {
  if (p == 1.f) return token_sum<LANES>(w);
  const float most = token_max<LANES>(w), a = w / most;   // NaN: in the lane's own term, or all are 0
  if (most == 0.f) return token_sum<LANES>(w);            // 0, or NaN
  const float sum = token_sum<LANES>(p == 2.f ? a * a : a == 0.f ? 0.f : powf(a, p));
  return most * (p == 2.f ? sqrtf(sum) : powf(sum, 1.f / p));
}

// A lane's R experts of a row.  WHOLE: rows and the base are whole pieces of R, a lane has R experts or none.
template <int DT, int R, bool WHOLE>
__device__ __forceinline__ void read_row(const typename Elem<DT>::type* __restrict__ row, int base, int experts, float past, float (&x)[R]) {
  typedef typename Elem<DT>::type E;
  if constexpr (WHOLE) {
    struct alignas(R * sizeof(E) < 16 ? R * sizeof(E) : 16) Piece { E v[R]; };
    Piece piece = {};
    if (base < experts) piece = *(const Piece*)(row + base);
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = base < experts ? Elem<DT>::to_f32(piece.v[r]) : past;
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float v = Elem<DT>::to_f32(row[base + r < experts ? base + r : experts - 1]);   // one load after the other, no branches
      x[r] = base + r < experts ? v : past;
    }
  }
}
template <int DT, int R, bool WHOLE>
__device__ __forceinline__ void write_row(typename Elem<DT>::type* __restrict__ row, int base, int experts, const float (&x)[R]) {
  typedef typename Elem<DT>::type E;
  if constexpr (WHOLE) {
    struct alignas(R * sizeof(E) < 16 ? R * sizeof(E) : 16) Piece { E v[R]; };
    Piece piece;
#pragma unroll
    for (int r = 0; r < R; ++r) piece.v[r] = Elem<DT>::from_f32(x[r]);
    if (base < experts) *(Piece*)(row + base) = piece;
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (base + r < experts) row[base + r] = Elem<DT>::from_f32(x[r]);
  }
}

// The largest logit of a token and the sum of exp(x - m), which the caller's e gets
template <int DT, int LANES, int R>
__device__ __forceinline__ void softmax_parts(const float (&x)[R], float& m, float& sum, float (&e)[R]) {
  m = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) m = fmaxf(m, x[r]);
  m = token_max<LANES>(m);
  sum = 0.f;
  // past the last expert x is -inf and adds nothing; of a token whose logits are all -inf the sum is not a number, as it should be
#pragma unroll
  for (int r = 0; r < R; ++r) {
    e[r] = exp_of<DT>(x[r] - m);
    sum += e[r];
  }
  sum = token_sum<LANES>(sum);
}

template <int DT> __device__ __forceinline__ float sigmoid_of(float x) { return over<DT>(1.f, 1.f + exp_of<DT>(-x)); }

// A token's choice again by the whole wave, with keys in 64 bits: lane j gets the j-th.
template <int DT, int R>
__device__ __forceinline__ int pick_wide(const typename Elem<DT>::type* __restrict__ row, const Choose& c) {
  const int lane = lane_id(), base = lane * R;
  double x[R], s[R];
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = base + r < c.experts ? (double)Elem<DT>::to_f32(row[base + r]) : (double)-INFINITY;
  if (c.sigmoid) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 1. / (1. + exp(-x[r]));
  } else {
    double sum = 0, top = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) top = larger(top, x[r]);
    top = token_max<64>(top);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = exp(x[r] - top);
      sum += s[r];
    }
    sum = token_sum<64>(sum);
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] /= sum;
  }
  if (c.bias) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] += base + r < c.experts ? (double)c.bias[base + r] : 0.;
  }
  uint64_t key[R];
  order_keys<R, false>(key, s, base, c.experts);
  if (c.top_groups < c.groups) {
    bool close;
    const uint64_t open = open_groups<64, R, double>(key, c, lane, close);
    if (!c.bias) order_keys<R, false>(key, x, base, c.experts);
    keep_open(key, open, base, c.experts / c.groups);
  }
  int mine = 0, next;
  pick<64, R>(key, lane, c.top_k, c.top_k, mine, next);
  return mine;
}

template <int DT, int LANES, int R, bool WHOLE>
__device__ __forceinline__ void choose_token(const float (&x)[R], const typename Elem<DT>::type* __restrict__ row, int64_t t, bool real, const Choose& c) {
  typedef typename Elem<DT>::type E;
  const int lane = lane_id() % LANES, base = lane * R, size = c.experts / c.groups;
  const bool grouped = c.top_groups < c.groups;
  // the uniform conditions stay outside of the loops over a lane's experts: inside they become a branch for each
  float m = 0.f, sum = 1.f, s[R];
  if (!c.sigmoid || c.lse) {
    softmax_parts<DT, LANES, R>(x, m, sum, s);
    if (c.lse) {
      float lse = m + logf(sum);
      if (__any(m == INFINITY || m == -INFINITY)) {     // the largest is none of the logits that are not numbers, which the sum then does not show
        float bad = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) bad = x[r] != x[r] ? 1.f : bad;
        bad = token_max<LANES>(bad);
        lse = bad != 0.f ? NAN : m == INFINITY || m == -INFINITY ? m : lse;
      }
      if (lane == 0 && real) c.lse[t] = lse;
    }
  }
  if (c.sigmoid) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = sigmoid_of<DT>(x[r]);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = over<DT>(s[r], sum);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (c.scores && real) write_row<DT, R, WHOLE>((E*)c.scores + t * c.experts, base, c.experts, s);

  uint32_t key[R];
  bool close = false;
  int mine = 0, next = -1;
  const int more = c.bias && c.top_k < c.top_groups * size ? 1 : 0;
  if (c.bias) {
    float bias[R];
    read_row<MBX_F32, R, WHOLE>(c.bias, base, c.experts, 0.f, bias);
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] += bias[r];
  }
  __builtin_amdgcn_sched_barrier(0);   // the parts one after the other: all at once take more registers than there are
  // without a bias a group goes by its scores where two are added up, else by its best logit, exactly as the choice does
  const bool by_score = c.bias || (grouped && c.group_best == 2);
  if (by_score) order_keys<R, WHOLE>(key, s, base, c.experts);
  else order_keys<R, WHOLE>(key, x, base, c.experts);
  if (grouped) {
    const uint64_t open = open_groups<LANES, R, float>(key, c, lane, close);
    close = close && by_score;
    if (by_score && !c.bias) order_keys<R, WHOLE>(key, x, base, c.experts);
    keep_open(key, open, base, size);
  }
  pick<LANES, R>(key, lane, c.top_k, c.top_k + more, mine, next);

  const bool live = lane < c.top_k;
  const auto score_of = [&](float logit) { return c.sigmoid ? sigmoid_of<DT>(logit) : over<DT>(exp_of<DT>(logit - m), sum); };
  if (c.bias) {
    // each chosen key against the next in the order, of the next lane or behind the last
    const int last = live ? mine : 0;
    const float x0 = Elem<DT>::to_f32(row[last]), b0 = c.bias[last], k0 = score_of(x0) + b0;
    float x1 = __shfl_down(x0, 1, LANES), b1 = __shfl_down(b0, 1, LANES), k1 = __shfl_down(k0, 1, LANES);
    if (lane == c.top_k - 1 && more) {
      x1 = Elem<DT>::to_f32(row[next]);
      b1 = c.bias[next];
      k1 = score_of(x1) + b1;
    }
    const bool twins = x0 == x1 && b0 == b1, border = lane == c.top_k - 1 && more;
    if (lane < c.top_k - 1 + more) close = close || (!(k0 - k1 > kCloseKeys * (1.f + fabsf(k0))) && !twins);
    // Twins on either side of the border say nothing of the keys behind them: the last chosen one against the largest left that is no twin of it.  16-bit logits and
    // equal biases make some tokens in a hundred such (32768 tokens, 8 of 256 experts, biases of zero: 20.9 us without this, 22.0 with it)
    if (__any(border && twins)) {
      const float x_last = __shfl(x0, c.top_k - 1, LANES), b_last = __shfl(b0, c.top_k - 1, LANES);
      float left[R], bias[R];
      read_row<DT, R, WHOLE>(row, base, c.experts, -INFINITY, left);
      read_row<MBX_F32, R, WHOLE>(c.bias, base, c.experts, 0.f, bias);
      uint32_t best = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) best = larger(best, left[r] == x_last && bias[r] == b_last ? 0 : key[r]);
      best = token_max<LANES>(best);
      if (border && twins && best != 0) close = close || !(k0 - unordered(best) > kCloseKeys * (1.f + fabsf(k0)));
    }
  }
  for (uint64_t left = __ballot(close); left != 0;) {
    const int first = __builtin_ctzll(left) & ~(LANES - 1);      // a token's lanes
    left &= LANES == 64 ? 0 : ~(0xffffull << first);
    const uint64_t at = (uint64_t)row;
    const uint64_t of = (uint64_t)(uint32_t)lane_value((int)(uint32_t)(at >> 32), first) << 32 | (uint32_t)lane_value((int)(uint32_t)at, first);
    const int wide = pick_wide<DT, (R * LANES + 63) / 64>((const E*)of, c);
    const int moved = __shfl(wide, lane);
    mine = (lane_id() & ~(LANES - 1)) == first ? moved : mine;
  }

  float w = live ? score_of(Elem<DT>::to_f32(row[mine])) : 0.f;
  if (c.norm_p > 0.f) {
    const float norm = token_pnorm<LANES>(w, c.norm_p);
    w = norm == 0.f ? 0.f : w / norm;   // scores that are all zero: weights of zero
  }
  if (live && real) {
    ((E*)c.weights)[t * c.top_k + lane] = Elem<DT>::from_f32(w * c.scale);
    c.indices[t * c.top_k + lane] = mine;
    if (c.indices32) c.indices32[t * c.top_k + lane] = mine;
  }
}

template <int DT, int LANES, int R, bool WHOLE>
__global__ void __launch_bounds__(kChooseThreads, 4) choose_kernel(const Choose c) {
  typedef typename Elem<DT>::type E;
  // no loop over tokens: what does not change in it would take registers all the time
  const int64_t token = c.first + (int64_t)blockIdx.x * (kChooseThreads / LANES) + threadIdx.x / LANES, t = token < c.tokens ? token : c.tokens - 1;
  const E* const row = (const E*)c.logits + t * c.experts;     // all lanes stay: the last token again, not written
  float x[R];
  read_row<DT, R, WHOLE>(row, lane_id() % LANES * R, c.experts, -INFINITY, x);
  choose_token<DT, LANES, R, WHOLE>(x, row, t, token < c.tokens, c);
}

// grad_logits from the gradients of weights, scores and lse (each may be NULL), in fp32 from the logits, by the gradient g of log s: nothing is divided by
// scores, which may be the smallest numbers there are
//   y = scale u, u = w / ||w||_p:   g = grad_scores s, + scale (dy u - (sum dy u) u^p) at the chosen experts, zero where the norm is;  without a norm + scale dy w
//   dx = g (1 - s) (sigmoid), g - s sum g (softmax);  + grad_lse softmax(x)
template <int DT, int LANES, int R, bool WHOLE>
__global__ void __launch_bounds__(kChooseThreads, 4)
choose_backward_kernel(const Choose c, const void* __restrict__ grad_weights, const void* __restrict__ grad_scores, const float* __restrict__ grad_lse,
                       void* __restrict__ grad_logits) {
  typedef typename Elem<DT>::type E;
  const int lane = lane_id() % LANES, base = lane * R;
  const int64_t token = c.first + (int64_t)blockIdx.x * (kChooseThreads / LANES) + threadIdx.x / LANES, t = token < c.tokens ? token : c.tokens - 1;
  const E* const row = (const E*)c.logits + t * c.experts;
  float x[R], g[R], soft[R], dx[R];
  read_row<DT, R, WHOLE>(row, base, c.experts, -INFINITY, x);
  if (grad_scores) read_row<DT, R, WHOLE>((const E*)grad_scores + t * c.experts, base, c.experts, 0.f, g);
  else {
#pragma unroll
    for (int r = 0; r < R; ++r) g[r] = 0.f;
  }
  float m = 0.f, sum = 1.f;
  if (!c.sigmoid || grad_lse) {
    softmax_parts<DT, LANES, R>(x, m, sum, soft);
#pragma unroll
    for (int r = 0; r < R; ++r) soft[r] = over<DT>(soft[r], sum);
  }
  if (c.sigmoid) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // s and 1 - s from exp(-|x|): exact towards either end
      const float a = exp_of<DT>(-fabsf(x[r])), b = over<DT>(1.f, 1.f + a);
      g[r] *= x[r] < 0.f ? a * b : b;
      dx[r] = x[r] < 0.f ? b : a * b;
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) g[r] *= soft[r];
  }
  if (grad_weights) {
    const bool live = lane < c.top_k;
    int mine = live ? (int)c.indices[t * c.top_k + lane] : 0;
    mine = mine < 0 || mine >= c.experts ? 0 : mine;
    float u = 0.f, dy = 0.f;
    if (live) {
      const float logit = Elem<DT>::to_f32(row[mine]);
      u = c.sigmoid ? sigmoid_of<DT>(logit) : over<DT>(exp_of<DT>(logit - m), sum);
      dy = Elem<DT>::to_f32(((const E*)grad_weights)[t * c.top_k + lane]) * c.scale;
    }
    float here;
    if (c.norm_p > 0.f) {
      const float p = c.norm_p, n = token_pnorm<LANES>(u, p);
      u = n == 0.f ? 0.f : u / n;
      here = dy * u - token_sum<LANES>(dy * u) * (p == 1.f ? u : p == 2.f ? u * u : u == 0.f ? 0.f : powf(u, p));
    } else {
      here = dy * u;
    }
    for (int j = 0; j < c.top_k; ++j) {
      const int e = __shfl(mine, j, LANES);
      const float v = __shfl(here, j, LANES);
#pragma unroll
      for (int r = 0; r < R; ++r) g[r] += base + r == e ? v : 0.f;
    }
  }
  if (c.sigmoid) {
#pragma unroll
    for (int r = 0; r < R; ++r) dx[r] *= g[r];
  } else {
    float dot = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) dot += g[r];
    dot = token_sum<LANES>(dot);
#pragma unroll
    for (int r = 0; r < R; ++r) dx[r] = g[r] - soft[r] * dot;
  }
  if (grad_lse) {
    const float of = grad_lse[t];
#pragma unroll
    for (int r = 0; r < R; ++r) dx[r] += of * soft[r];
  }
  if (token < c.tokens) write_row<DT, R, WHOLE>((E*)grad_logits + t * c.experts, base, c.experts, dx);
}

// bias + rate sign(mean count - count), the mean in whole numbers: of every layer a workgroup.
constexpr int kBalanceLayers = 64;
template <int MOST>
struct Balance {
  const float* bias[MOST];
  const int32_t* counts[MOST];
  float* out[MOST];
  int rows[MOST];
};

template <int MOST>
__global__ void __launch_bounds__(kChooseThreads) balance_kernel(const Balance<MOST> layers, int experts, float rate) {
  __shared__ int64_t sums[kChooseThreads / kWave];
  const float* const bias = layers.bias[blockIdx.x];
  const int32_t* const counts = layers.counts[blockIdx.x];
  float* const out = layers.out[blockIdx.x];
  const int rows = layers.rows[blockIdx.x];
  const auto count_of = [&](int e) {
    int64_t n = 0;
    for (int row = 0; row < rows; ++row) n += counts[(int64_t)row * experts + e];
    return n;
  };
  int64_t total = 0;
  for (int e = threadIdx.x; e < experts; e += kChooseThreads) total += count_of(e);
  total = over_token<64>(total, [](int64_t a, int64_t b) { return a + b; });
  if (lane_id() == 0) sums[threadIdx.x / kWave] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kChooseThreads / kWave; ++w) total += sums[w];
  for (int e = threadIdx.x; e < experts; e += kChooseThreads) {
    const int64_t off = total - count_of(e) * experts;
    out[e] = bias[e] + (off > 0 ? rate : off < 0 ? -rate : 0.f);
  }
}

template <int MOST>
static void launch_balance(const float* const* bias, const int32_t* const* counts, const int* rows, float* const* out, int layers, int experts, float rate,
                           hipStream_t s) {
  Balance<MOST> of = {};
  for (int l = 0; l < layers; ++l) {
    of.bias[l] = bias[l];
    of.counts[l] = counts[l];
    of.out[l] = out[l];
    of.rows[l] = rows[l];
  }
  balance_kernel<MOST><<<(unsigned)layers, kChooseThreads, 0, s>>>(of, experts, rate);
}

constexpr int64_t kChooseMaxBlocks = 1 << 23;   // of a launch, whose threads have to be fewer than 2^32

// 16 lanes a token take fewer instructions a token; of more than 64 experts 64 lanes have the shorter way to the end, which counts until there are a few
// waves for every SIMD: 8 of 256 experts, groups and bias, of 1 / 1024 / 4096 / 32768 tokens 7.7 / 12.6 / 13.3 / 27.6 us with 16 lanes, 5.9 / 10.6 / 13.4 /
// 44.8 us with 64 (6 of 64 experts: 3.5 / 3.9 / 4.1 / 8.6 and 3.4 / 3.8 / 4.9 / 18.9).
static bool few_lanes(const Choose& c) {
  return c.experts <= 256 && c.top_k <= 16 && c.groups <= 16 && (c.experts <= 64 || c.tokens > 2048);
}

static bool pieces(const Choose& c, int r, int size, const void* a, const void* b, const void* d) {
  const uintptr_t at = (uintptr_t)a | (uintptr_t)b | (uintptr_t)d, piece = (uintptr_t)(r * size < 16 ? r * size : 16);
  return c.experts % r == 0 && at % piece == 0 && (uintptr_t)c.bias % (uintptr_t)(r * 4 < 16 ? r * 4 : 16) == 0;
}

// KERNEL<DT, LANES, R, WHOLE> of the sizes
#define MBX_CHOOSE_LANES(KERNEL, DT, LANES, R, SIZE, A, B, D, ...)                                                                            \
  for (constexpr int kTokens = kChooseThreads / LANES; c.first < tokens; c.first += kChooseMaxBlocks * kTokens) {                             \
    const unsigned grid = (unsigned)smaller<int64_t>(kChooseMaxBlocks, ceil_div(tokens - c.first, kTokens));                                  \
    if (pieces(c, R, SIZE, A, B, D)) KERNEL<DT, LANES, R, true><<<grid, kChooseThreads, 0, s>>>(__VA_ARGS__);                                 \
    else KERNEL<DT, LANES, R, false><<<grid, kChooseThreads, 0, s>>>(__VA_ARGS__);                                                            \
  }
#define MBX_CHOOSE(DT, KERNEL, SIZE, A, B, D, ...)                                                                                            \
  do {                                                                                                                                        \
    if (few_lanes(c)) {                                                                                                                       \
      if (c.experts <= 16) { MBX_CHOOSE_LANES(KERNEL, DT, 16, 1, SIZE, A, B, D, __VA_ARGS__) }                                                  \
      else if (c.experts <= 32) { MBX_CHOOSE_LANES(KERNEL, DT, 16, 2, SIZE, A, B, D, __VA_ARGS__) }                                             \
      else if (c.experts <= 64) { MBX_CHOOSE_LANES(KERNEL, DT, 16, 4, SIZE, A, B, D, __VA_ARGS__) }                                             \
      else if (c.experts <= 128) { MBX_CHOOSE_LANES(KERNEL, DT, 16, 8, SIZE, A, B, D, __VA_ARGS__) }                                            \
      else { MBX_CHOOSE_LANES(KERNEL, DT, 16, 16, SIZE, A, B, D, __VA_ARGS__) }                                                                 \
    } else {                                                                                                                                  \
      if (c.experts <= 64) { MBX_CHOOSE_LANES(KERNEL, DT, 64, 1, SIZE, A, B, D, __VA_ARGS__) }                                                  \
      else if (c.experts <= 128) { MBX_CHOOSE_LANES(KERNEL, DT, 64, 2, SIZE, A, B, D, __VA_ARGS__) }                                            \
      else if (c.experts <= 256) { MBX_CHOOSE_LANES(KERNEL, DT, 64, 4, SIZE, A, B, D, __VA_ARGS__) }                                            \
      else { MBX_CHOOSE_LANES(KERNEL, DT, 64, 8, SIZE, A, B, D, __VA_ARGS__) }                                                                  \
    }                                                                                                                                         \
  } while (0)

static int choose_sizes(int dtype, int64_t tokens, int experts, int top_k, int score, int groups, int top_groups, int group_best, float norm_p, float scale) {
  if (dtype != MBX_BF16 && dtype != MBX_F16 && dtype != MBX_F32) return MBX_EINVAL;
  if (tokens < 0 || experts <= 0 || top_k <= 0 || (score != MBX_SCORE_SOFTMAX && score != MBX_SCORE_SIGMOID)) return MBX_EINVAL;
  if (groups <= 0 || experts % groups || top_groups <= 0 || top_groups > groups || (group_best != 1 && group_best != 2)) return MBX_EINVAL;
  if ((int64_t)top_k > (int64_t)top_groups * (experts / groups) || !(norm_p >= 0.f) || !(norm_p < INFINITY) || !(scale - scale == 0.f)) return MBX_EINVAL;
  if (experts > kChooseMaxExperts || top_k > kChooseMaxTopK || groups > kChooseMaxGroups) return MBX_EUNSUPPORTED;
  if (tokens > 0x7fffffff) return MBX_ERANGE;
  return 0;
}

}  // namespace
}  // namespace mbx

using namespace mbx;

extern "C" {

int mbx_choose_experts(const void* logits, int dtype, int64_t tokens, int num_experts, int top_k, int score, const float* bias, int groups, int top_groups,
                       int group_best, float norm_p, float scale, void* scores, void* weights, int64_t* indices, int32_t* indices32, float* lse,
                       mbx_stream_t stream) {
  const int rc = choose_sizes(dtype, tokens, num_experts, top_k, score, groups, top_groups, group_best, norm_p, scale);
  if (rc || tokens == 0) return rc;
  if (!logits || !weights || !indices) return MBX_EINVAL;
  Choose c = {logits, bias, tokens, num_experts, top_k, score == MBX_SCORE_SIGMOID, groups, top_groups, group_best, norm_p, scale,
                    scores, weights, indices, indices32, lse, 0};
  hipStream_t s = as_stream(stream);
  if (dtype == MBX_BF16) MBX_CHOOSE(MBX_BF16, choose_kernel, 2, logits, scores, nullptr, c);
  else if (dtype == MBX_F16) MBX_CHOOSE(MBX_F16, choose_kernel, 2, logits, scores, nullptr, c);
  else MBX_CHOOSE(MBX_F32, choose_kernel, 4, logits, scores, nullptr, c);
  return launch_status();
}

int mbx_choose_experts_backward(const void* grad_weights, const void* grad_scores, const float* grad_lse, const void* logits, const int64_t* indices, int dtype,
                                int64_t tokens, int num_experts, int top_k, int score, float norm_p, float scale, void* grad_logits, mbx_stream_t stream) {
  const int rc = choose_sizes(dtype, tokens, num_experts, top_k, score, 1, 1, 1, norm_p, scale);
  if (rc || tokens == 0) return rc;
  if (!logits || !grad_logits || (grad_weights && !indices)) return MBX_EINVAL;
  Choose c = {logits, nullptr, tokens, num_experts, top_k, score == MBX_SCORE_SIGMOID, 1, 1, 1, norm_p, scale,
                    nullptr, nullptr, const_cast<int64_t*>(indices), nullptr, nullptr, 0};
  hipStream_t s = as_stream(stream);
  if (dtype == MBX_BF16) MBX_CHOOSE(MBX_BF16, choose_backward_kernel, 2, logits, grad_scores, grad_logits, c, grad_weights, grad_scores, grad_lse, grad_logits);
  else if (dtype == MBX_F16) MBX_CHOOSE(MBX_F16, choose_backward_kernel, 2, logits, grad_scores, grad_logits, c, grad_weights, grad_scores, grad_lse, grad_logits);
  else MBX_CHOOSE(MBX_F32, choose_backward_kernel, 4, logits, grad_scores, grad_logits, c, grad_weights, grad_scores, grad_lse, grad_logits);
  return launch_status();
}

int mbx_balance_bias(const float* const* bias, const int32_t* const* counts, const int* rows, float* const* out, int layers, int num_experts, float rate,
                     mbx_stream_t stream) {
  if (layers < 0 || num_experts <= 0) return MBX_EINVAL;
  if (layers == 0) return 0;
  if (!bias || !counts || !rows || !out) return MBX_EINVAL;
  for (int l = 0; l < layers; ++l)
    if (!bias[l] || !out[l] || rows[l] < 0 || (rows[l] > 0 && !counts[l])) return MBX_EINVAL;
  hipStream_t s = as_stream(stream);
  if (layers == 1) launch_balance<1>(bias, counts, rows, out, 1, num_experts, rate, s);
  else
    for (int first = 0; first < layers; first += kBalanceLayers)
      launch_balance<kBalanceLayers>(bias + first, counts + first, rows + first, out + first, layers - first < kBalanceLayers ? layers - first : kBalanceLayers,
                                     num_experts, rate, s);
  return launch_status();
}

}  // extern "C"
