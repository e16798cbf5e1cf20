// SPDX-License-Identifier: Apache-2.0
// What a row of logits says of a given token: its log probability and its rank, the
// row's entropy, and the first tokens of the order (logits descending, equal ones by
// index) with theirs.
//
// With m the largest logit and d = x - m, others = sum exp(d) over all tokens but one of
// the largest, t = sum d exp(d):
//   log p(x) = d - log1p(others),  entropy = log1p(others) - t / (1 + others).
// Without the largest token's own 1 in the sum, a row that is sure of its token keeps
// what is left of it: both terms have one sign, so neither cancels.
//
// A wave takes a segment of 2048 logits in registers, so it reads them once and knows
// its largest before it forms a weight. It leaves (m, sum, t, count of the largest) and
// the largest of each group of 64 logits. The first k tokens are then found top down: the
// first k segments, of their groups the first k, of these groups' logits the first k, each in
// order of (largest, index). (A token outside them has k segments or groups before it,
// each with a token that comes before it.) So the row is not read again but for k groups,
// and segments whose sum needs exact weights.
// Vocabularies up to 2048 need one wave a row and one launch.
//
// What bounds it. 256 rows of 131072 BF16 logits (67 MB, 13.3 us of a copy): segments
// 19.4 us, 3.5 TB/s, between bytes and vector instructions (15 a logit, the vector units
// active half of the cycles: conversion, maximum, an exponential, the two sums, and a
// wave's reductions; segments of 4096 logits take 125 registers and 3.5 us more); join 5.7 us.
// 8192 rows of 512 F32 logits (17 MB, 3.4 us): 11.6 us in one round of waves, each a chain
// of reductions; four rows a wave measured 13.7. One row, or 5 rows of 100003: launches and
// chains of loads, 4.0 us, and 6.5 + 8.1 with 20 alternatives.
#include "common.hpp"
#include "lanes.hpp"
#include "ops.hpp"

#include <cmath>

namespace evo::hip {

namespace {

constexpr uint32_t kNoToken = 0xffffffffU;
constexpr int kSegment = 2048, kGroup = 64, kGroups = kSegment / kGroup;
constexpr int kMostTop = 64;

// Of one segment: its largest logit, how many are equal to it, and the sums of exp(d)
// and of d exp(d) over the others. before: tokens in front of the given one.
struct Segment {
  float top, sum, spread;
  uint32_t equal, before, unused[3];
};

struct LogprobArgs {
  const void *logits;
  int rows, vocab, segments;
  size_t row_stride;
  const uint32_t *tokens;
  float *logprob;
  uint32_t *rank;
  float *entropy;
  int alternatives;
  uint32_t *top_tokens;
  float *top_logprobs;
  Segment *stats;  // [rows][segments]
  float *groups;   // [rows][segments * kGroups], the largest of each
};

__device__ inline float value_of_order(uint32_t order) {
  return __builtin_bit_cast(float, (order & 0x80000000U) != 0 ? order & 0x7fffffffU : ~order);
}
// A token's place: larger is earlier.
__device__ inline uint64_t place(uint32_t order, uint32_t index) {
  return static_cast<uint64_t>(order) << 32 | ~index;
}
__device__ inline uint32_t order_of(uint64_t place) { return static_cast<uint32_t>(place >> 32); }
__device__ inline uint32_t index_of(uint64_t place) { return ~static_cast<uint32_t>(place); }

// kPer logits a lane, in runs of kEach: 16 bytes, wherever a row starts (the loads need no
// alignment), or one. Every lane loads from inside its row: a run that would pass its end
// is moved back to it, and what came twice or lies behind it is -infinity.
template <typename S, int kRun, int kPer> struct Logits {
  static constexpr int kEach = kRun;
  float x[kPer];

  // Where run i / kEach of a lane begins in a row, and where it is loaded from.
  static __device__ int begin(int first, int i) {
    return first + (i / kEach * 64 + static_cast<int>(threadIdx.x & 63)) * kEach;
  }
  static __device__ int from(int first, int i, int vocab) {
    return min(begin(first, i), vocab - kEach);
  }
  // Logits first .. of a row (vocab >= kEach), and the given token's among all of them,
  // whose load follows the token's own and would wait alone behind theirs.
  __device__ float load(const S *row, int first, int vocab, uint32_t token) {
    typedef S vector __attribute__((ext_vector_type(kEach)));
    typedef vector unaligned __attribute__((aligned(sizeof(S))));
    unaligned v[kPer / kEach];
#pragma unroll
    for (int i = 0; i < kPer; i += kEach)
      v[i / kEach] = *reinterpret_cast<const unaligned *>(row + from(first, i, vocab));
    const S given = row[token < static_cast<uint32_t>(vocab) ? token : 0];
    asm volatile("" ::: "memory");  // every load before the first use
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      x[i] = static_cast<float>(v[i / kEach][i % kEach]);
    if (first + kPer * 64 > vocab) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[i] = valid(first, i, vocab) ? x[i] : -INFINITY;
    }
    return static_cast<float>(given);
  }
  static __device__ bool valid(int first, int i, int vocab) {
    return i % kEach >= begin(first, i) - from(first, i, vocab);
  }
};

// (fmaxf would quiet each operand first.)
__device__ inline float largest(float x, float y, float z) {
  float most;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(most) : "v"(x), "v"(y), "v"(z));
  return most;
}
__device__ inline float larger(float x, float y) { return __builtin_fmaxf(x, y); }
template <int kCtrl> __device__ inline float largest_with(float x) {
  const float other = dpp<kCtrl, 0xf>(x, x);
  return largest(x, other, other);
}
template <int kCount> __device__ inline float largest_of(const float *x) {
  if constexpr (kCount == 1)
    return x[0];
  else if constexpr (kCount == 2)
    return largest(x[0], x[1], x[1]);
  else
    return largest(largest_of<kCount - 2>(x), x[kCount - 2], x[kCount - 1]);
}

constexpr float kLog2e = 1.44269504088896341F, kLog2eLow = 1.92596299e-8F;
constexpr float kLn2 = 0.693147180559945F;
// exp(d) for d <= 0 with its argument's rounding, up to |d| * 2^-24, added again.
__device__ inline float exact_weight(float d) {
  const float scaled = d * kLog2e;
  const float w = __builtin_amdgcn_exp2f(scaled);
  const float lost = fmaf(d, kLog2eLow, fmaf(d, kLog2e, -scaled));
  // (-infinity leaves no number.)
  return w == 0.0F ? 0.0F : fmaf(w * lost, kLn2, w);
}

// The sums of a segment, given the largest of each kChunk registers. A chunk without the
// largest of all in any lane takes the short way: with base * kLog2e = high + low, a
// weight is exp2(x kLog2e - high), and 2^-low comes in at the end. (What log2(e) has beyond
// kLog2e is left out of both products, so an exponent lacks |x - base| 2^-25.6, less than its
// rounding to F32 may take; in low alone it would be a factor of 2^(base 2^-25.6).)
constexpr int kChunk = 8;
template <int kPer>
__device__ inline void sums(const float (&x)[kPer], const float (&most)[kPer / kChunk],
                            Segment &s) {
  const float base = s.top == -INFINITY ? 0.0F : s.top;
  const float high = base * kLog2e;
  const float low = fmaf(base, kLog2e, -high);
  float sum = 0.0F, spread = 0.0F, short_sum = 0.0F, short_spread = 0.0F;
  uint32_t equal = 0;
#pragma unroll
  for (int i = 0; i < kPer; i += kChunk) {
    if (__any(most[i / kChunk] == base)) {
#pragma unroll
      for (int e = 0; e < kChunk; ++e) {
        const bool first = x[i + e] == base;
        const float d = x[i + e] - base;
        const float w = first ? 0.0F : __builtin_amdgcn_exp2f(d * kLog2e);
        equal += first ? 1U : 0U;
        sum += w;
        spread = fmaf(w, larger(d, -200.0F), spread);  // (a weight of 0 has d = -infinity)
      }
    } else {
#pragma unroll
      for (int e = 0; e < kChunk; ++e) {
        const float scaled = fmaf(x[i + e], kLog2e, -high), w = __builtin_amdgcn_exp2f(scaled);
        short_sum += w;
        short_spread = fmaf(w, larger(scaled, -300.0F), short_spread);
      }
    }
  }
  const float lift = __builtin_amdgcn_exp2f(-low);
  s.sum = wave_reduce(fmaf(short_sum, lift, sum), Sum());
  s.spread = wave_reduce(fmaf((short_spread - low * short_sum) * lift, kLn2, spread), Sum());
  s.equal = wave_reduce(equal, Sum());
}
// The same with exact weights, of kPer logits a lane at a time.
struct ExactSums {
  float base, sum = 0.0F, spread = 0.0F;
  uint32_t equal = 0;
  __device__ explicit ExactSums(float top) : base(top == -INFINITY ? 0.0F : top) {}
  template <int kPer> __device__ void add(const float (&x)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = x[i] - base, w = x[i] == base ? 0.0F : exact_weight(d);
      equal += x[i] == base ? 1U : 0U;
      sum += w;
      spread = fmaf(w, larger(d, -200.0F), spread);
    }
  }
  __device__ void finish(Segment &s) const {
    s.sum = wave_reduce(sum, Sum());
    s.spread = wave_reduce(spread, Sum());
    s.equal = wave_reduce(equal, Sum());
  }
};

// Largest logit and sums of a segment, which x holds; every lane has them. Sums of a small
// total come from far logits, whose arguments round worst: they are formed again, exactly,
// from logits that are read again (kept for that, they would cost every wave registers).
// So are those of logits whose multiple by log2(e) might overflow. (No weight at all is
// exact: segments of masked logits are not read again, 256 x 131072 of which all but 100 a row
// are -infinity 32 us for 41.)
template <typename S, int kPer>
__device__ inline Segment segment_of(const S *row, int first, int vocab, const float (&x)[kPer],
                                     const float (&most)[kPer / kChunk]) {
  Segment s{};
  s.top = wave_reduce(largest_of<kPer / kChunk>(most), Most());
  const bool large = fabsf(s.top) > 0x1p120F && s.top != -INFINITY;
  if (!large)
    sums(x, most, s);
  if (large || (!(s.sum >= 0.0625F) && s.sum != 0.0F)) {
    ExactSums exact(s.top);
#pragma unroll 1
    for (int i = first + static_cast<int>(threadIdx.x & 63); i < first + 64 * kPer; i += 64 * 8) {
      float again[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        again[j] = static_cast<float>(row[min(i + 64 * j, vocab - 1)]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        again[j] = i + 64 * j < vocab ? again[j] : -INFINITY;
      exact.add(again);
    }
    exact.finish(s);
  }
  return s;
}

// Tokens of the segment in front of `token`, whose logit is `given`.
template <typename L, int kPer>
__device__ inline uint32_t count_before(const float (&x)[kPer], const float (&most)[kPer / kChunk],
                                        int first, int vocab, float given, int token) {
  // Those behind it in the row come before it only by a larger logit.
  const float above = value_of_order(ordered(given) + 1);
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < kPer; i += kChunk) {
    if (!__any(most[i / kChunk] >= given))
      continue;
#pragma unroll
    for (int j = i; j < i + kChunk; j += L::kEach) {
      const int from = L::from(first, j, vocab);
      // (What stands in for a logit that came twice, -infinity, comes before no token.)
      if (__any((from <= token && token < from + L::kEach) || from != L::begin(first, j))) {
#pragma unroll
        for (int e = 0; e < L::kEach; ++e) {
          const bool ahead = from + e < token && L::valid(first, j + e, vocab);
          count += __popcll(__ballot(x[j + e] >= (ahead ? given : above)));
        }
      } else {
        const float least = from < token ? given : above;
#pragma unroll
        for (int e = 0; e < L::kEach; ++e)
          count += __popcll(__ballot(x[j + e] >= least));
      }
    }
  }
  return count;
}

// A row's results from its whole sums.
struct Row {
  float top, log_total, entropy;
  bool valid;  // a row with a logit above -infinity, and none that is NaN or +infinity
  __device__ explicit Row(const Segment &s) : top(s.top) {
    const float others = static_cast<float>(s.equal - 1) + s.sum;
    valid = s.top > -INFINITY && s.top < INFINITY && s.sum == s.sum;
    log_total = log1pf(others);
    entropy = log_total - s.spread / (1.0F + others);
  }
  __device__ float logprob(float logit) const {
    return valid ? logit - top - log_total : __builtin_nanf("");
  }
};
__device__ inline void write_row(const LogprobArgs &a, int row, const Row &r, uint32_t before,
                                 bool given, float logit) {
  if (a.logprob != nullptr)
    a.logprob[row] = given ? r.logprob(logit) : __builtin_nanf("");
  if (a.rank != nullptr)
    a.rank[row] = given && r.valid ? before : kNoToken;
  if (a.entropy != nullptr)
    a.entropy[row] = r.valid ? r.entropy : __builtin_nanf("");
}
__device__ inline void write_top(const LogprobArgs &a, int row, const Row &r, int rank,
                                 uint64_t place) {
  const size_t at = static_cast<size_t>(row) * a.alternatives + rank;
  a.top_tokens[at] = index_of(place);
  a.top_logprobs[at] = r.logprob(value_of_order(order_of(place)));
}
// The alternatives of a row without them. (Its NaN are in no order that a search could follow:
// one may stand for a maximum or not, and the order of some is 0, that of no token.)
__device__ inline void write_no_top(const LogprobArgs &a, int row) {
  const int lane = threadIdx.x & 63;
  if (lane < a.alternatives) {
    const size_t at = static_cast<size_t>(row) * a.alternatives + lane;
    a.top_tokens[at] = kNoToken;
    a.top_logprobs[at] = __builtin_nanf("");
  }
}

// A value that k of the wave's lanes reach, and with one less few more (0: fewer lanes have
// any): a few from the top down, more by the bits of it (8192 x 512, us with 1, 4 and 10
// alternatives: 10.0, 11.1 and 12.6, by bits 11.0, 11.5 and 12.0).
__device__ inline uint32_t reached_by(uint32_t mine, int k) {
  uint32_t border = 0;
  if (k <= 8) {
#pragma unroll 1
    for (int count = 0; count < k;) {
      border = wave_reduce(mine, Most());
      if (border == 0)
        break;
      const bool first = mine == border;
      count += __popcll(__ballot(first));
      mine = first ? 0 : mine;
    }
    return border;
  }
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t tried = border | 1U << bit;
    const int count = __popcll(__ballot(mine >= tried));
    if (count >= k)
      border = tried;
    if (count == k)
      break;
  }
  return border;
}
// The k largest of n different places in LDS, moved to the list's beginning in any
// order; returns how many (n, if there are no more). One wave calls it.
__device__ inline int keep_best(uint64_t *list, int n, int k) {
  const int lane = threadIdx.x & 63;
  wave_sync();
  if (n <= k)
    return n;
  uint64_t border = 0;
#pragma unroll 1
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t tried = border | uint64_t{1} << bit;
    int count = 0;
    for (int i = 0; i < n; i += 64)
      count += __popcll(__ballot(i + lane < n && list[i + lane] >= tried));
    if (count >= k)
      border = tried;
    if (count == k)
      break;
  }
  int kept = 0;
  for (int i = 0; i < n; i += 64) {
    const uint64_t own = i + lane < n ? list[i + lane] : 0;
    const uint64_t in = __ballot(own >= border && i + lane < n);
    if (in >> lane & 1)
      list[kept + __popcll(in & ((uint64_t{1} << lane) - 1))] = own;
    kept += __popcll(in);
  }
  wave_sync();
  return kept;
}
// Writes the first tokens of a row, which are among n places. One wave calls it.
__device__ inline void write_best(const LogprobArgs &a, int row, const Row &r,
                                  const uint64_t *list, int n) {
  const int lane = threadIdx.x & 63;
  wave_sync();
#pragma unroll 1
  for (int first = 0; first < n; first += 64) {
    const uint64_t own = first + lane < n ? list[first + lane] : 0;
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i)
      rank += list[i] > own ? 1 : 0;
    if (first + lane < n && rank < a.alternatives)
      write_top(a, row, r, rank, own);
  }
}

// ------------------------------------------------- one wave takes a row
// The first tokens of a row that a wave holds; list: 64 * kPer places.
template <typename L, int kPer>
__device__ inline void first_tokens(const LogprobArgs &a, int row, const Row &r,
                                    const float (&x)[kPer], uint64_t *list) {
  const int lane = threadIdx.x & 63, k = a.alternatives;
  // The k-th largest of the lanes' largest (0: fewer lanes have one) bounds the k-th
  // token from below.
  uint32_t order[kPer], most = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    order[i] = L::valid(0, i, a.vocab) ? ordered(x[i]) : 0;
    most = max(most, order[i]);
  }
  uint32_t border = max(reached_by(most, k), 1U);
  int n = 0;
#pragma unroll 1
  for (bool closer = false;; closer = true) {
    n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t in = __ballot(order[i] >= border);
      if (in == 0)
        continue;
      if (in >> lane & 1)
        list[n + __popcll(in & ((uint64_t{1} << lane) - 1))] =
            place(order[i], static_cast<uint32_t>(L::from(0, i, a.vocab) + i % L::kEach));
      n += __popcll(in);
    }
    if (n <= 64 || closer)
      break;
    // Where k is about the number of lanes, that bound is far from the k-th token: one that
    // leaves at most 64 is looked for among all (1024 rows of 512, 64 alternatives: 10 us for
    // 22 with the places themselves). Only equal logits may leave more.
    uint32_t found = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t tried = found | 1U << bit;
      int count = n;
      if (tried > border) {
        count = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          count += __popcll(__ballot(order[i] >= tried));
      }
      if (count >= k)
        found = tried;
      if (count >= k && count <= 64)
        break;
    }
    border = max(border, found);
  }
  if (n > 256)
    n = keep_best(list, n, k);
  write_best(a, row, r, list, n);
}

template <typename S, int kRun, int kPer>
__global__ __launch_bounds__(256) void row_kernel(const LogprobArgs a) {
  typedef Logits<S, kRun, kPer> L;
  extern __shared__ uint64_t lists[];  // [4][64 * kPer], where alternatives are asked for
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + wave;
  if (row >= a.rows)
    return;
  const S *logits = static_cast<const S *>(a.logits) + row * a.row_stride;
  const uint32_t token = a.tokens != nullptr ? a.tokens[row] : kNoToken;
  L l;
  const float logit = l.load(logits, 0, a.vocab, token);
  const bool given = token < static_cast<uint32_t>(a.vocab);
  float chunks[kPer / kChunk];
#pragma unroll
  for (int i = 0; i < kPer; i += kChunk)
    chunks[i / kChunk] = largest_of<kChunk>(&l.x[i]);
  Segment s{};
  s.top = wave_reduce(largest_of<kPer / kChunk>(chunks), Most());
  // (As segment_of: exact weights alone took 9.5 us for 8.2, 1024 rows of 2000.)
  const bool large = fabsf(s.top) > 0x1p120F && s.top != -INFINITY;
  if (!large)
    sums(l.x, chunks, s);
  if (large || (!(s.sum >= 0.0625F) && s.sum != 0.0F)) {
    ExactSums exact(s.top);
    exact.add(l.x);
    exact.finish(s);
  }
  if (given && a.rank != nullptr)
    s.before = count_before<L>(l.x, chunks, 0, a.vocab, logit, static_cast<int>(token));
  const Row r(s);
  if (lane == 0)
    write_row(a, row, r, s.before, given, logit);
  if (a.alternatives > 0 && r.valid)
    first_tokens<L>(a, row, r, l.x, lists + wave * (64 * kPer));
  else
    write_no_top(a, row);
}

// ------------------------------------------------- rows of several segments
template <typename S> __global__ __launch_bounds__(256) void segment_kernel(const LogprobArgs a) {
  typedef Logits<S, 16 / static_cast<int>(sizeof(S)), kSegment / 64> L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const unsigned at = blockIdx.x * 4 + wave;
  const int row = static_cast<int>(at / a.segments), segment = static_cast<int>(at % a.segments);
  if (row >= a.rows)
    return;
  const S *logits = static_cast<const S *>(a.logits) + row * a.row_stride;
  const uint32_t token = a.tokens != nullptr && a.rank != nullptr ? a.tokens[row] : kNoToken;
  const int first = segment * kSegment;
  L l;
  const float logit = l.load(logits, first, a.vocab, token);
  const bool given = token < static_cast<uint32_t>(a.vocab);

  // The largest of each run, of 8 registers and of 64 neighbours: kEach registers in each
  // of 64 / kEach lanes.
  constexpr int kPer = kSegment / 64, kLanes = kGroup / L::kEach, kRuns = kPer / L::kEach;
  float chunks[kPer / kChunk], mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; i += kChunk) {
    float runs[kChunk / L::kEach];
#pragma unroll
    for (int j = 0; j < kChunk / L::kEach; ++j)
      runs[j] = largest_of<L::kEach>(&l.x[i + j * L::kEach]);
    chunks[i / kChunk] = largest_of<kChunk / L::kEach>(runs);
    if (a.alternatives > 0) {
#pragma unroll
      for (int j = 0; j < kChunk / L::kEach; ++j) {
        float most = largest_with<0xb1>(runs[j]);  // quad_perm 1 0 3 2
        most = largest_with<0x4e>(most);           // quad_perm 2 3 0 1
        most = largest_with<0x141>(most);          // row_half_mirror
        if constexpr (kLanes == 16)
          most = largest_with<0x140>(most);  // row_mirror
        mine = lane % kLanes == i / L::kEach + j ? most : mine;
      }
    }
  }
  if (a.alternatives > 0 && lane % kLanes < kRuns)
    a.groups[(static_cast<size_t>(row) * a.segments + segment) * kGroups +
             lane % kLanes * (64 / kLanes) + lane / kLanes] = mine;
  Segment s = segment_of(logits, first, a.vocab, l.x, chunks);
  if (given && s.top >= logit)
    s.before = count_before<L>(l.x, chunks, first, a.vocab, logit, static_cast<int>(token));
  if (lane == 0)
    a.stats[at] = s;
}

// The k best and at most 256 of n places, n up to 4096, to `best`; returns how many. All
// threads of the block call it. Where every lane has places, each wave finds the border that
// k / 4 of its lanes' largest reach, and the lowest of the four has k above it; with fewer
// places, the highest of those that k of a wave's reach (0: no wave has so many) does.
// The counter is its own: waves that are late may still read it when others, behind no
// barrier, begin the next list.
__device__ inline int filter(uint64_t *list, int n, int k, uint64_t *best) {
  __shared__ uint32_t borders[4];
  __shared__ int found;
  const int lane = threadIdx.x & 63;
  uint32_t most = 0;
  for (int i = threadIdx.x; i < n; i += 256)
    most = max(most, order_of(list[i]));
  const bool all = n >= 256;
  const int wanted = all ? (k + 3) / 4 : k;
  uint32_t border = reached_by(most, wanted);
  if (lane == 0)
    borders[threadIdx.x >> 6] = border;
  if (threadIdx.x == 0)
    found = 0;
  __syncthreads();
  border = all ? min(min(borders[0], borders[1]), min(borders[2], borders[3]))
               : max(max(borders[0], borders[1]), max(borders[2], borders[3]));
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t own = list[i];
    if (order_of(own) >= border) {
      const int at = atomicAdd(&found, 1);
      if (at < 256)
        best[at] = own;
    }
  }
  __syncthreads();
  if (found <= 256)
    return found;
  // (Many equal logits.)
  if (threadIdx.x < 64) {
    const int kept = keep_best(list, n, k);
    if (lane < kept)
      best[lane] = list[lane];
  }
  __syncthreads();
  return min(n, k);
}

// A row's segments joined, and its first tokens.
template <typename S> __global__ __launch_bounds__(256) void join_kernel(const LogprobArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t list[kMostTop * kGroup];
  __shared__ __attribute__((aligned(16))) uint64_t fewer[256];
  __shared__ uint32_t chosen[kMostTop];
  __shared__ int count;
  __shared__ uint32_t least;
  static_assert(kGroups <= kGroup, "groups of the best segments fit the list");
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const Segment *stats = a.stats + static_cast<size_t>(row) * a.segments;
  const S *logits = static_cast<const S *>(a.logits) + row * a.row_stride;
  const uint32_t token = a.tokens != nullptr ? a.tokens[row] : kNoToken;
  const bool given = token < static_cast<uint32_t>(a.vocab);
  const int k = a.alternatives;

  // Every wave joins the sums by itself.
  Segment whole{}, own{};
  whole.top = own.top = -INFINITY;
  if (lane < a.segments)
    own = stats[lane];
  for (int i = lane; i < a.segments; i += 64) {
    const float top = i < 64 ? own.top : stats[i].top;
    whole.top = larger(whole.top, top);
    if (k > 0 && threadIdx.x < 64)
      list[i] = place(ordered(top), static_cast<uint32_t>(i));
  }
  // (After the first statistics, which would wait for the token.)
  const float logit = given ? static_cast<float>(logits[token]) : 0.0F;
  whole.top = wave_reduce(whole.top, Most());
  for (int i = lane; i < a.segments; i += 64) {
    const Segment s = i < 64 ? own : stats[i];
    whole.before += s.before;
    if (s.top == whole.top) {
      whole.equal += s.equal;
      whole.sum += s.sum;
      whole.spread += s.spread;
    } else {
      // (Nothing above -infinity: its sum is zero, or NaN.)
      const float away = larger(s.top - whole.top, -200.0F), shrink = expf(s.top - whole.top);
      const float sum = s.sum + (s.top == -INFINITY ? 0.0F : static_cast<float>(s.equal));
      whole.sum += shrink * sum;
      whole.spread += shrink * fmaf(away, sum, s.spread);
    }
  }
  whole.sum = wave_reduce(whole.sum, Sum());
  whole.spread = wave_reduce(whole.spread, Sum());
  whole.equal = wave_reduce(whole.equal, Sum());
  whole.before = wave_reduce(whole.before, Sum());
  const Row r(whole);
  if (threadIdx.x == 0)
    write_row(a, row, r, whole.before, given, logit);
  if (k == 0)
    return;
  if (!r.valid) {  // (All waves find the same.)
    if (threadIdx.x < 64)
      write_no_top(a, row);
    return;
  }

  // Each round takes the k best of the list (all, if there are no more) in order: of the
  // segments, their groups, and those groups' logits. What waves share is written a barrier
  // after its last reads: fewer, chosen, least, count and what filter shares behind the one
  // that begins a round, the list behind the one in its middle.
  int n = a.segments;
#pragma unroll 1
  for (int round = 0;; ++round) {
    __syncthreads();
    const uint64_t *from = list;
    if (n > 128) {  // (Ranks take n steps, the threshold about 32: 184 x 17449 41 -> 16 us.)
      from = fewer;
      n = filter(list, n, k, fewer);
    }
    const int kept = min(n, k);
    if (static_cast<int>(threadIdx.x) < n) {
      const uint64_t mine = from[threadIdx.x];
      int rank = 0;
#pragma unroll 16
      for (int i = 0; i < n; ++i)
        rank += from[i] > mine ? 1 : 0;
      if (rank < kept && round == 2)
        write_top(a, row, r, rank, mine);
      if (rank < kept)
        chosen[rank] = index_of(mine);
      if (rank == kept - 1)
        least = order_of(mine);
    }
    if (round == 2)
      return;
    if (threadIdx.x == 0)
      count = 0;
    __syncthreads();
    // What lies below the k-th of these is below k tokens.
    const uint32_t border = kept < k ? 0 : least;
    const int each = round == 0 ? kGroups : kGroup;
    for (int i = threadIdx.x; i < kept * each; i += 256) {
      const uint32_t index = chosen[i / each] * each + i % each;
      uint32_t order = 0;
      if (round == 0 && index * kGroup < static_cast<uint32_t>(a.vocab))
        order = ordered(a.groups[static_cast<size_t>(row) * a.segments * kGroups + index]);
      else if (round == 1 && index < static_cast<uint32_t>(a.vocab))
        order = ordered(static_cast<float>(logits[index]));
      if (order != 0 && order >= border)
        list[atomicAdd(&count, 1)] = place(order, index);
    }
    __syncthreads();
    n = count;
  }
}

template <typename S, int kRun, int kPer>
void launch_rows(const LogprobArgs &a, hipStream_t stream) {
  const size_t lists = a.alternatives > 0 ? 4 * 64 * kPer * sizeof(uint64_t) : 0;
  hipLaunchKernelGGL((row_kernel<S, kRun, kPer>), dim3(ceil_div(a.rows, 4)), dim3(256),
                     static_cast<unsigned>(lists), stream, a);
}

template <typename S> void launch(const LogprobArgs &a, hipStream_t stream) {
  constexpr int kRun = 16 / static_cast<int>(sizeof(S));
  if (a.vocab < kRun)
    return launch_rows<S, 1, 8>(a, stream);
  if (a.vocab <= 512)
    return launch_rows<S, kRun, 8>(a, stream);
  if (a.vocab <= 1024)
    return launch_rows<S, kRun, 16>(a, stream);
  if (a.vocab <= kSegment)
    return launch_rows<S, kRun, 32>(a, stream);
  const size_t waves = static_cast<size_t>(a.rows) * a.segments;
  hipLaunchKernelGGL(segment_kernel<S>, dim3(ceil_div(waves, 4)), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(join_kernel<S>, dim3(a.rows), dim3(256), 0, stream, a);
}

constexpr size_t kMostRows = size_t{1} << 20;
size_t segments_of(size_t vocab) { return (vocab + kSegment - 1) / kSegment; }
// Waves of segment_kernel that its launch takes, four a block: it counts threads in 32 bits.
constexpr size_t kMostSegments = ((size_t{1} << 32) - 1) / 256 * 4;

}  // namespace

size_t token_logprobs_workspace_bytes(size_t rows, size_t vocab, size_t alternatives) {
  if (rows > kMostRows || vocab > kMostRows || vocab <= kSegment ||
      rows * segments_of(vocab) > kMostSegments)
    return 0;
  return rows * segments_of(vocab) *
         (sizeof(Segment) + (alternatives > 0 ? kGroups * sizeof(float) : 0));
}

Status token_logprobs(int dtype, const void *logits, size_t rows, size_t vocab, size_t row_stride,
                      const uint32_t *tokens, float *logprob, uint32_t *rank, float *entropy,
                      size_t alternatives, uint32_t *top_tokens, float *top_logprobs,
                      void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (dtype != kElementF32 && dtype != kElementBF16 && dtype != kElementF16)
    return {ErrorCode::kInvalidArgument, "token_logprobs: logits are F32, BF16 or F16"};
  const size_t size = dtype == kElementF32 ? 4 : 2;
  if (logits == nullptr || rows == 0 || rows > kMostRows || vocab == 0 || vocab > kMostRows ||
      row_stride < vocab || row_stride > (size_t{1} << 40) ||
      reinterpret_cast<uintptr_t>(logits) % size != 0)
    return {ErrorCode::kInvalidArgument,
            "token_logprobs: rows, vocab or row_stride out of range, or misaligned logits"};
  const auto at = [](const void *tensor) { return reinterpret_cast<uintptr_t>(tensor); };
  if ((at(tokens) | at(logprob) | at(rank) | at(entropy) | at(top_tokens) | at(top_logprobs)) % 4)
    return {ErrorCode::kInvalidArgument, "token_logprobs: tokens or outputs not 4-byte aligned"};
  if (tokens == nullptr && (logprob != nullptr || rank != nullptr))
    return {ErrorCode::kInvalidArgument, "token_logprobs: logprob and rank need tokens"};
  if (alternatives > kMostTop || alternatives > vocab ||
      (alternatives > 0 && (top_tokens == nullptr || top_logprobs == nullptr)))
    return {ErrorCode::kInvalidArgument,
            "token_logprobs: at most 64 alternatives, no more than vocab, with their outputs"};
  if (logprob == nullptr && rank == nullptr && entropy == nullptr && alternatives == 0)
    return {ErrorCode::kInvalidArgument, "token_logprobs: no output"};
  const size_t segments = segments_of(vocab);
  if (rows * segments > kMostSegments)
    return {ErrorCode::kInvalidArgument, "token_logprobs: grid too large"};
  const size_t need = token_logprobs_workspace_bytes(rows, vocab, alternatives);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return {ErrorCode::kInvalidArgument, "token_logprobs: workspace too small or not aligned"};
  Segment *const stats = static_cast<Segment *>(workspace);
  const LogprobArgs args{logits, static_cast<int>(rows), static_cast<int>(vocab),
                         static_cast<int>(segments), row_stride, tokens, logprob, rank, entropy,
                         static_cast<int>(alternatives), top_tokens, top_logprobs, stats,
                         need > 0 ? reinterpret_cast<float *>(stats + rows * segments) : nullptr};
  if (dtype == kElementF32)
    launch<float>(args, stream);
  else if (dtype == kElementBF16)
    launch<__bf16>(args, stream);
  else
    launch<_Float16>(args, stream);
  return launch_status("token_logprobs kernels");
}

}  // namespace evo::hip
