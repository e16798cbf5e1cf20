// SPDX-License-Identifier: Apache-2.0
// One token per row of logits: temperature, top-k, nucleus (top-p), min-p and
// a given uniform draw, over the order of evo_sampler_sample: logits
// descending, equal ones by index.
//
// Every cut keeps a beginning of that order, and the draw takes the first token
// whose cumulative weight passes uniform * (weight kept), so no row is sorted: a
// histogram over the order (counts and weights) tells which bin holds each
// border, and only that bin's tokens are ranked.
//
// The weights exp((logit - top) / temperature) are 64-bit and summed as
// integers of 2^-B: such a sum has no order, so neither the atomics of the
// histogram nor a split of a row can change a token. B = 63 - ceil(log2(vocab)),
// 51 at most, is what 64-bit sums leave room for: each weight is rounded by up to
// 2^-(B+1) of the largest, so a border is off by vocab * 2^-(B+1) at most (512
// values 1.1e-13, 131072 9.3e-10, 2^20 6.0e-8). A weight below 2^-(B+1) counts as
// none.
//
// A row is read two or three times. Every index and every loop is bounded whatever
// the later reads find, so that logits or a workspace that someone else writes
// meanwhile cost the row its token and no more.
//
// What bounds it: 2048 rows of 512 values 10.4 us, one round of waves, each a chain of
// reductions, LDS atomics and two or three searches; 128 rows of 131072 BF16 values 64
// us, of which their ranges take 7.6 (34 MB, 4.4 TB/s),
// the histograms 21 (the weights' 64-bit arithmetic), and the borders 35 (a block a row:
// 13 to read the row again for the borders' bins, the rest scans and searches of one
// wave after another).
#include "common.hpp"
#include "lanes.hpp"
#include "ops.hpp"

#include <algorithm>
#include <cmath>

namespace evo::hip {

namespace {

constexpr uint32_t kNoToken = 0xffffffffU;

struct SampleArgs {
  const void *logits;
  int vocab;
  size_t row_stride;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p, *uniform;
  uint32_t *tokens;
  double units;  // 2^B, the largest weight
  double reach;  // exp(-reach) = 2^-(B+2)
};

// Place of a token in the order: larger is earlier. 56 bits, vocab <= 2^20.
__device__ inline uint64_t place(float v, int index) {
  return static_cast<uint64_t>(ordered(v)) << 24 | static_cast<uint32_t>(0xffffff - index);
}

__device__ inline uint32_t token_of(uint64_t place) {
  return place == 0 ? kNoToken : 0xffffffU - static_cast<uint32_t>(place & 0xffffff);
}
__device__ inline float value_of(uint64_t place) {
  const uint32_t bits = static_cast<uint32_t>(place >> 24);
  return __builtin_bit_cast(float, (bits & 0x80000000U) != 0 ? bits & 0x7fffffffU : ~bits);
}

// 2^(i / 64).
__device__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// exp(x) in units of 2^-B, B <= 51, rounded, for x = z * ln(2) / 64 in [-37, 0]: with
// z = n + f, 2^(n / 64) from a table and a shift, exp(f ln(2) / 64) by its
// series to the fifth power in f (the next term is below 2^-54).
__device__ inline uint64_t weight_units(double z, const double *powers) {
  const double n = __builtin_rint(z), f = z - n;
  double e = 1.2417843701716925e-12;
  e = fma(e, f, 5.7328516886404019e-10);
  e = fma(e, f, 2.1173137155464776e-07);
  e = fma(e, f, 5.86490495505617e-05);
  e = fma(e, f, 0.010830424696249145);
  e = fma(e, f, 1.0);
  // powers[] is the table times 2^B; whole / 64 goes into the exponent.
  const int whole = static_cast<int>(n);
  const uint64_t bits = __builtin_bit_cast(uint64_t, e * powers[whole & 63]) +
                        (static_cast<uint64_t>(static_cast<uint32_t>(whole & ~63) << 14) << 32);
  // Adding 2^52 rounds to a whole number in the low bits.
  const double shifted = __builtin_bit_cast(double, bits) + 4503599627370496.0;
  return __builtin_bit_cast(uint64_t, shifted) - 0x4330000000000000ULL;
}

// A row's parameters.
struct Cuts {
  float temperature, top_p, min_p, uniform;
  int top_k;
  double units;
  __device__ Cuts(const SampleArgs &a, size_t r)
      : temperature(a.temperature == nullptr ? 1.0F : a.temperature[r]),
        top_p(a.top_p == nullptr ? 1.0F : a.top_p[r]),
        min_p(a.min_p == nullptr ? 0.0F : a.min_p[r]), uniform(a.uniform[r]),
        top_k(a.top_k == nullptr ? 0 : a.top_k[r]), units(a.units) {}
  __device__ bool valid() const {
    return temperature >= 0.0F && temperature < INFINITY && top_k >= 0 && top_p > 0.0F &&
           top_p <= 1.0F && min_p >= 0.0F && min_p <= 1.0F && uniform == uniform;
  }
  // Whether a row of this largest logit can be sampled.
  __device__ bool samples(float top) const { return valid() && top < INFINITY && top > -INFINITY; }
  __device__ bool has_k(int vocab) const { return top_k > 0 && top_k < vocab; }
  __device__ bool greedy() const { return temperature == 0.0F || top_k == 1; }
  // Least weight that min-p keeps.
  __device__ uint64_t least() const {
    return static_cast<uint64_t>(__builtin_ceil(static_cast<double>(min_p) * units));
  }
  // The nucleus keeps tokens while the weight before them is below top_p * total: up
  // to the first at which the weight, itself included, passes this.
  __device__ uint64_t nucleus(uint64_t total) const {
    const uint64_t reach = static_cast<uint64_t>(
        __builtin_ceil(static_cast<double>(top_p) * static_cast<double>(total)));
    return (reach < total ? reach : total) - 1;
  }
  // The draw takes the first token at which the weight passes this.
  __device__ uint64_t draw(uint64_t total) const {
    const double drawn = fmax(static_cast<double>(uniform), 0.0) * static_cast<double>(total);
    if (drawn >= static_cast<double>(total))
      return total - 1;
    const uint64_t whole = static_cast<uint64_t>(drawn);
    return whole < total ? whole : total - 1;
  }
};

// Values low <= v < high.
struct Values {
  float low, high;
  __device__ bool has(float v) const { return v >= low && v < high; }
  // Their places, the first in order and the last.
  __device__ uint64_t first() const {
    return high == INFINITY ? ~0ULL : (static_cast<uint64_t>(ordered(high)) << 24) - 1;
  }
  __device__ uint64_t last() const { return static_cast<uint64_t>(ordered(low)) << 24; }
};

// How a row's values map to bins and weights, given its largest and lowest value.
struct Scale {
  float top, reach, bin_scale;
  int last_bin;
  double unit;  // 64 / (ln 2 * temperature)
  __device__ Scale(const SampleArgs &a, float top_, float low, float temperature, int bins)
      : top(top_), reach(static_cast<float>(
                       fmin(a.reach * static_cast<double>(temperature), 3.0e38))),
        last_bin(bins - 1),
        unit(92.33248261893106 / static_cast<double>(temperature)) {
    const float range = fminf(reach, top - low);
    // A little less than bins / range: the last value stays inside.
    bin_scale = range > 0.0F ? fminf(static_cast<float>(bins) * 0.999999F / range, 3.0e38F) : 0.0F;
  }
  // Bin of a value, -1 for one without weight. Every step is monotonic, so a bin is a
  // range of values.
  __device__ int bin(float v) const {
    const float below = top - v;
    return below <= reach ? min(static_cast<int>(below * bin_scale), last_bin) : -1;
  }
  // Lowest value of the bins 0 .. `bin`: the 64 values around the one that the bin's
  // end maps back to are tried, then, 64 at a time, all. All lanes of a wave call it,
  // with the same bin.
  __device__ float lowest(int bin) const {
    const float end = static_cast<float>(bin + 1);
    const auto inside = [&](uint64_t key) {
      const float v = value_of(key << 24);
      return key >= 0xff800000U || ((top - v) * bin_scale < end && top - v <= reach);
    };
    const uint64_t lane = threadIdx.x & 63;
    uint64_t below = ordered(fmaxf(top - end / bin_scale, -3.0e38F)) - 33;
    const uint64_t tried = __ballot(inside(below + lane));
    if (tried != 0 && (tried & 1) == 0) {
      below += __builtin_ctzll(tried) - 1;
    } else {
      below = 0x007fffffU;  // -infinity, in no bin
#pragma unroll 1
      for (int shift = 26; shift >= 0; shift = shift == 2 ? 0 : shift - 6) {
        const uint64_t in = __ballot(inside(below + ((lane + 1) << shift)));
        below += static_cast<uint64_t>(in == 0 ? 64 : __builtin_ctzll(in)) << shift;
      }
    }
    return value_of((below + 1) << 24);
  }
  __device__ Values values(int first, int last) const {  // of a run of bins
    return {lowest(last), first == 0 ? INFINITY : lowest(first - 1)};
  }
  __device__ uint64_t weight(float v, const double *powers) const {  // of one in reach
    return weight_units((static_cast<double>(v) - static_cast<double>(top)) * unit, powers);
  }
};

// ------------------------------------------------------- one wave's search
// 256 bins of counts and weights in LDS, four a lane.
struct WaveBins {
  uint64_t *mass;
  uint32_t *count;
  __device__ void clear() const {
    const int lane = threadIdx.x & 63;
    reinterpret_cast<uint4 *>(mass)[2 * lane] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(mass)[2 * lane + 1] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(count)[lane] = make_uint4(0, 0, 0, 0);
    wave_sync();
  }
  __device__ void add(int bin, uint64_t w) const {
    atomicAdd(&count[bin], 1U);
    atomicAdd(reinterpret_cast<unsigned long long *>(&mass[bin]),
              static_cast<unsigned long long>(w));
  }
};
// The lane's four bins, and what lies before them.
struct LaneBins {
  uint64_t mass[4], mass_before, mass_total;
  uint32_t count[4], count_before, count_total;
  __device__ explicit LaneBins(const WaveBins &bins) {
    const int lane = threadIdx.x & 63;
    wave_sync();
    uint64_t m = 0;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mass[j] = bins.mass[4 * lane + j];
      count[j] = bins.count[4 * lane + j];
      m += mass[j];
      c += count[j];
    }
    const uint64_t own_m = m;
    const uint32_t own_c = c;
    m = wave_scan<Sum>(m);
    c = wave_scan<Sum>(c);
    mass_before = m - own_m;
    count_before = c - own_c;
    mass_total = lane_value(m, 63);
    count_total = lane_value(c, 63);
  }
};
// The bin in which the running count or weight passes a target, what lies before it,
// and how many tokens it has.
struct Hit {
  int bin;
  uint64_t mass_before;
  uint32_t count_before, members;
};
__device__ inline Hit locate(const LaneBins &b, bool by_count, uint64_t target) {
  uint64_t at_m = b.mass_before;
  uint32_t at_c = b.count_before;
  Hit h{-1, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t from = by_count ? at_c : at_m;
    const uint64_t size = by_count ? b.count[j] : b.mass[j];
    if (target >= from && target - from < size)
      h = {4 * static_cast<int>(threadIdx.x & 63) + j, at_m, at_c, b.count[j]};
    at_m += b.mass[j];
    at_c += b.count[j];
  }
  const uint64_t owner = __ballot(h.bin >= 0);
  const int from = owner == 0 ? 0 : __builtin_ctzll(owner);
  return Hit{lane_value(h.bin, from), lane_value(h.mass_before, from),
             lane_value(h.count_before, from), lane_value(h.members, from)};
}

// Among the tokens that the lanes hold (spot[e] != 0: a place; w[e]: its weight;
// `members` of them), the one, in order, at which the running count or weight passes
// the target: its place; `before` grows by the weight up to it, itself included. A
// histogram over the range of the places leaves the few that are taken one by one: seven
// of them at most, as each leaves eight of 56 bits less. 0 where there is none.
template <int kPer>
__device__ inline uint64_t wave_find(uint64_t (&spot)[kPer], const uint64_t (&w)[kPer],
                                     uint32_t members, const WaveBins &bins, bool by_count,
                                     uint64_t target, uint64_t &before) {
  for (int pass = 0; members > 6 && pass < 7; ++pass) {
    uint64_t last = ~0ULL, first = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      first = first > spot[e] ? first : spot[e];
      last = spot[e] != 0 && spot[e] < last ? spot[e] : last;
    }
    first = wave_reduce(first, Most{});
    last = wave_reduce(last, Least{});
    const int shift = max(0, 56 - static_cast<int>(__builtin_clzll(first - last)));
    bins.clear();
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (spot[e] != 0)
        bins.add(static_cast<int>((first - spot[e]) >> shift), w[e]);
    const Hit h = locate(LaneBins(bins), by_count, target);
    before += h.mass_before;
    target -= by_count ? h.count_before : h.mass_before;
    members = h.members;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (spot[e] != 0 && static_cast<int>((first - spot[e]) >> shift) != h.bin)
        spot[e] = 0;
  }
  uint64_t token = 0;
  for (uint32_t i = 0; i < members; ++i) {
    uint64_t first = 0, own = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      own = spot[e] > first ? w[e] : own;
      first = spot[e] > first ? spot[e] : first;
    }
    token = wave_reduce(first, Most{});
    own = lane_value(own, __builtin_ctzll(__ballot(first == token)));
    before += own;
    if (by_count ? target == i : target < own)
      break;
    target -= by_count ? 0 : own;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      spot[e] = spot[e] == token ? 0 : spot[e];
  }
  return token;
}

// ------------------------------------------------------- small vocabularies
// A wave per row, kPer values a lane in registers.
template <typename T, int kPer>
__global__ __launch_bounds__(64) void sample_wave_kernel(const SampleArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t mass_s[256];
  __shared__ __attribute__((aligned(16))) uint32_t count_s[256];
  __shared__ double powers[64];
  const int lane = threadIdx.x;
  const size_t r = blockIdx.x;
  const T *logits = static_cast<const T *>(a.logits) + r * a.row_stride;
  float v[kPer];  // value e of the lane is token 64 * e + lane
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    v[e] = 64 * e + lane < a.vocab ? static_cast<float>(logits[64 * e + lane]) : -INFINITY;
  const Cuts cuts(a, r);
  powers[lane] = kPowers[lane] * a.units;
  const WaveBins bins{mass_s, count_s};
  bins.clear();
  float top = -INFINITY, low = INFINITY;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    bad |= !(v[e] < INFINITY);
    top = fmaxf(top, v[e]);
    low = 64 * e + lane < a.vocab ? fminf(low, v[e]) : low;
  }
  top = wave_reduce(top, Most{});
  low = wave_reduce(low, Least{});
  if (__any(bad) || !cuts.samples(top)) {
    if (lane == 0)
      a.tokens[r] = kNoToken;
    return;
  }
  if (cuts.greedy()) {
    int first = a.vocab;
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e)
      first = v[e] == top ? 64 * e + lane : first;
    first = wave_reduce(first, Least{});
    if (lane == 0)
      a.tokens[r] = static_cast<uint32_t>(first);
    return;
  }
  const Scale scale(a, top, low, cuts.temperature, 256);
  uint64_t w[kPer], kept = 0;
  int bin[kPer];
  const uint64_t least = cuts.least();
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    bin[e] = scale.bin(v[e]);
    w[e] = bin[e] >= 0 ? scale.weight(v[e], powers) : 0;
    kept += w[e] >= least ? w[e] : 0;
    if (bin[e] >= 0)
      bins.add(bin[e], w[e]);
  }
  const LaneBins all(bins);
  // The top-k border, the nucleus' border, the draw: one after the other through the
  // same code (three copies of it cost more to fetch than to run).
  uint64_t total = all.mass_total, token = 0;
#pragma unroll 1
  for (int border = 0; border < 3; ++border) {
    uint64_t target;
    if (border == 0) {
      if (cuts.top_k == 0 || static_cast<uint32_t>(cuts.top_k) >= all.count_total)
        continue;
      target = static_cast<uint64_t>(cuts.top_k) - 1;
    } else if (border == 1) {
      if (cuts.top_p >= 1.0F)
        continue;
      target = cuts.nucleus(total);
    } else {
      if (cuts.min_p > 0.0F) {
        kept = wave_reduce(kept, Sum{});
        total = Least{}(total, kept);
      }
      target = cuts.draw(total);
    }
    const Hit h = locate(all, border == 0, target);
    uint64_t spot[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      spot[e] = bin[e] == h.bin ? place(v[e], 64 * e + lane) : 0;
    total = h.mass_before;
    token = wave_find<kPer>(spot, w, h.members, bins, border == 0,
                            target - (border == 0 ? h.count_before : h.mass_before), total);
  }
  if (lane == 0)
    a.tokens[r] = token_of(token);
}

// ------------------------------------------------------- large vocabularies
template <typename T> struct Row {  // or a part of one, from token `first`
  const T *logits;
  int vocab, first;
  bool vector;  // it starts on 16 bytes
  __device__ Row(const SampleArgs &a, size_t r, int first_, int count)
      : logits(static_cast<const T *>(a.logits) + r * a.row_stride + first_), vocab(count),
        first(first_), vector(reinterpret_cast<uintptr_t>(logits) % 16 == 0) {}
  // f(value, index) over the tokens, 16 bytes a load where the row is aligned, kLoads
  // of them at a time and as many ahead. kLoads 1 where f is long: code of more copies
  // is fetched more slowly than it runs; 4 where it is short and the loads are what
  // takes the time.
  static constexpr int kPer = 16 / sizeof(T);
  typedef T wide __attribute__((ext_vector_type(16 / sizeof(T))));
  template <int kThreads, int kLoads>
  __device__ void load(wide (&to)[kLoads], int c = threadIdx.x) const {
    const wide *src = reinterpret_cast<const wide *>(logits);
#pragma unroll
    for (int a = 0; a < kLoads; ++a)
      if (vector && c + a * kThreads < vocab / kPer)
        to[a] = src[c + a * kThreads];
  }
  template <int kThreads, int kLoads, typename F> __device__ void each(F &&f) const {
    wide now[kLoads];
    load<kThreads, kLoads>(now);
    each<kThreads, kLoads>(now, f);
  }
  // The same where the caller has called load() already, ahead of other waits.
  template <int kThreads, int kLoads, typename F>
  __device__ void each(wide (&now)[kLoads], F &&f) const {
    each_load<kThreads, kLoads>(
        now,
        [&](const auto &values, int i) {
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            f(static_cast<float>(values[e]), i + e);
        },
        f);
  }
  // And with whole(values of a load, index of the first) for the 16-byte loads.
  template <int kThreads, int kLoads, typename W, typename F>
  __device__ void each_load(wide (&now)[kLoads], W &&whole_load, F &&f) const {
    int tail = 0;
    if (vector) {
      const int whole = vocab / kPer;
      wide next[kLoads];
#pragma unroll 1
      for (int c = threadIdx.x; c < whole; c += kThreads * kLoads) {
        load<kThreads, kLoads>(next, c + kThreads * kLoads);
#pragma unroll
        for (int a = 0; a < kLoads; ++a)
          if (a == 0 || c + a * kThreads < whole)
            whole_load(now[a], first + (c + a * kThreads) * kPer);
#pragma unroll
        for (int a = 0; a < kLoads; ++a)
          now[a] = next[a];
      }
      tail = whole * kPer;
    }
#pragma unroll 1
    for (int i = tail + threadIdx.x; i < vocab; i += kThreads)
      f(static_cast<float>(logits[i]), first + i);
  }
};

// A row's histogram and a list of tokens.
constexpr int kFew = 512;  // tokens that one wave searches
template <int kThreads, int kBins, int kList> struct SampleShared {
  uint64_t mass[kBins];   // before the scan a bin's own, then of the bins before it
  uint32_t count[kBins];
  uint64_t list_place[kList], list_mass[kList];
  __attribute__((aligned(16))) uint64_t sub_mass[256];
  __attribute__((aligned(16))) uint32_t sub_count[256];
  uint64_t few_place[kFew], few_mass[kFew];
  uint64_t wave_mass[kThreads / 64];
  uint32_t wave_count[kThreads / 64];
  double powers[64];
  uint64_t found_place, found_mass;
  uint32_t fill;
};

// Exclusive scan of count and mass over `size` entries.
template <int kThreads>
__device__ inline void scan_bins(uint32_t *count, uint64_t *mass, int size, uint32_t *wave_count,
                                 uint64_t *wave_mass) {
  const int per = (size + kThreads - 1) / kThreads, first = threadIdx.x * per;
  uint32_t c = 0;
  uint64_t m = 0;
  for (int i = first; i < min(first + per, size); ++i) {
    c += count[i];
    m += mass[i];
  }
  const uint32_t own_c = c;
  const uint64_t own_m = m;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  c = wave_scan<Sum>(c);
  m = wave_scan<Sum>(m);
  if (lane == 63) {
    wave_count[wave] = c;
    wave_mass[wave] = m;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    c += wave_count[w];
    m += wave_mass[w];
  }
  c -= own_c;
  m -= own_m;
  for (int i = first; i < min(first + per, size); ++i) {
    const uint32_t next_c = count[i];
    const uint64_t next_m = mass[i];
    count[i] = c;
    mass[i] = m;
    c += next_c;
    m += next_m;
  }
  __syncthreads();
}

// Last entry of an ascending array that is <= target (the first is).
template <typename V> __device__ inline int last_at_most(const V *a, int size, V target) {
  int low = 0, high = size;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (a[middle] <= target)
      low = middle;
    else
      high = middle;
  }
  return low;
}

// Among the list's `size` tokens the `members` whose places lie in last .. first: the
// one, in order, at which their running count (by_count) or weight passes the target.
// Its place, and in *mass the weight up to it, itself included. More than one wave
// searches are narrowed by histograms over the range of their places.
template <int kThreads, int kBins, int kList>
__device__ inline uint64_t find_in_list(SampleShared<kThreads, kBins, kList> &s, uint32_t size,
                                        uint64_t last, uint64_t first, uint32_t members,
                                        bool by_count, uint64_t target, uint64_t *mass) {
  __shared__ uint64_t scratch[kThreads / 64];
  uint64_t before = 0;
  for (int pass = 0; members > kFew && pass < 7; ++pass) {
    uint64_t lo = ~0ULL, hi = 0;
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
      const uint64_t p = s.list_place[i];
      if (p >= last && p <= first) {
        lo = p < lo ? p : lo;
        hi = p > hi ? p : hi;
      }
    }
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.sub_count[i] = 0;
      s.sub_mass[i] = 0;
    }
    hi = block_reduce<kThreads>(hi, scratch, Most{});
    lo = block_reduce<kThreads>(lo, scratch, Least{});
    const int shift = max(0, 56 - static_cast<int>(__builtin_clzll(hi - lo)));
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
      const uint64_t p = s.list_place[i];
      if (p >= last && p <= first)
        WaveBins{s.sub_mass, s.sub_count}.add(static_cast<int>((hi - p) >> shift),
                                              s.list_mass[i]);
    }
    __syncthreads();
    scan_bins<kThreads>(s.sub_count, s.sub_mass, 256, s.wave_count, s.wave_mass);
    const int sub = by_count ? last_at_most(s.sub_count, 256, static_cast<uint32_t>(target))
                             : last_at_most(s.sub_mass, 256, target);
    const uint32_t ahead = s.sub_count[sub];
    members = (sub == 255 ? members : s.sub_count[sub + 1]) - ahead;
    before += s.sub_mass[sub];
    target -= by_count ? ahead : s.sub_mass[sub];
    first = hi - (static_cast<uint64_t>(sub) << shift);
    const uint64_t span = (uint64_t{1} << shift) - 1;
    last = first < span ? 0 : first - span;
    __syncthreads();
  }
  if (threadIdx.x == 0)
    s.fill = 0;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
    const uint64_t p = s.list_place[i];
    if (p >= last && p <= first) {
      const uint32_t slot = atomicAdd(&s.fill, 1U);
      if (slot < kFew) {
        s.few_place[slot] = p;
        s.few_mass[slot] = s.list_mass[i];
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    members = min(members, min(s.fill, static_cast<uint32_t>(kFew)));
    constexpr int kPer = kFew / 64;
    uint64_t spot[kPer], w[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint32_t i = 64 * e + threadIdx.x;
      spot[e] = i < members ? s.few_place[i] : 0;
      w[e] = i < members ? s.few_mass[i] : 0;
    }
    const uint64_t place = wave_find<kPer>(spot, w, members,
                                           WaveBins{s.sub_mass, s.sub_count}, by_count, target,
                                           before);
    if (threadIdx.x == 0) {
      s.found_place = place;
      s.found_mass = before;
    }
  }
  __syncthreads();
  *mass = s.found_mass;
  return s.found_place;
}

// Lists the tokens whose values lie in `one` or `other` and whose place begins with
// `prefix` above `shift` bits, and their weights. Returns how many the list holds.
template <typename T, int kThreads, int kBins, int kList>
__device__ inline uint32_t gather(const Row<T> &row, const Scale &scale,
                              SampleShared<kThreads, kBins, kList> &s, const Values &one,
                              const Values &other, int shift, uint64_t prefix) {
  if (threadIdx.x == 0)
    s.fill = 0;
  __syncthreads();
  const auto push = [&](int i) {
    if (shift < 56 && place(static_cast<float>(row.logits[i]), i) >> shift != prefix)
      return;
    const uint32_t slot = atomicAdd(&s.fill, 1U);
    if (slot < kList)  // (there are no more, unless someone writes the logits meanwhile)
      s.list_place[slot] = static_cast<uint64_t>(i);
  };
  const auto wanted = [&](float v) { return one.has(v) || other.has(v); };
  // Few of the tokens are wanted: a load's make a mask without a branch.
  typename Row<T>::wide now[4];
  row.template load<kThreads, 4>(now);
  row.template each_load<kThreads, 4>(
      now,
      [&](const auto &values, int i) {
        uint32_t mask = 0;
#pragma unroll
        for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e)
          mask |= wanted(static_cast<float>(values[e])) ? 1U << e : 0;
        for (; mask != 0; mask &= mask - 1)
          push(i + __builtin_ctz(mask));
      },
      [&](float v, int i) {
        if (wanted(v))
          push(i);
      });
  __syncthreads();
  const uint32_t held = min(s.fill, static_cast<uint32_t>(kList));
  for (uint32_t i = threadIdx.x; i < held; i += kThreads) {
    const int token = static_cast<int>(s.list_place[i]);
    const float v = static_cast<float>(row.logits[token]);
    s.list_place[i] = place(v, token);
    s.list_mass[i] = scale.weight(v, s.powers);
  }
  __syncthreads();
  return held;
}

// Lists the `members` tokens of a bin, or, where they are more than the list holds,
// those of them among which the target is passed; members, target and the weight
// before them follow. Returns how many the list holds.
template <typename T, int kThreads, int kBins, int kList>
__device__ inline uint32_t list_bin(const Row<T> &row, const Scale &scale,
                                SampleShared<kThreads, kBins, kList> &s, int bin,
                                bool by_count, uint32_t &members, uint64_t &target,
                                uint64_t &before) {
  // Tokens whose place begins with `prefix` in its bits above `shift`.
  uint64_t prefix = 0;
  int shift = 56;
  const Values values = scale.values(bin, bin);
  while (members > kList && shift > 0) {
    // More than the list holds (many equal logits): 8 bits of the place at a time.
    shift -= 8;
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.sub_count[i] = 0;
      s.sub_mass[i] = 0;
    }
    __syncthreads();
    row.template each<kThreads, 1>([&](float v, int i) {
      if (!values.has(v))
        return;
      const uint64_t p = place(v, i);
      if (p >> (shift + 8) != prefix)
        return;
      const int digit = 255 - static_cast<int>((p >> shift) & 255);  // earlier first
      atomicAdd(&s.sub_count[digit], 1U);
      atomicAdd(reinterpret_cast<unsigned long long *>(&s.sub_mass[digit]),
                static_cast<unsigned long long>(scale.weight(v, s.powers)));
    });
    __syncthreads();
    scan_bins<kThreads>(s.sub_count, s.sub_mass, 256, s.wave_count, s.wave_mass);
    // Equal entries: the last of them is the one with tokens behind it.
    const int digit = by_count
                          ? last_at_most(s.sub_count, 256, static_cast<uint32_t>(target))
                          : last_at_most(s.sub_mass, 256, target);
    const uint32_t ahead = s.sub_count[digit];
    members = (digit == 255 ? members : s.sub_count[digit + 1]) - ahead;
    before += s.sub_mass[digit];
    target -= by_count ? ahead : s.sub_mass[digit];
    prefix = prefix << 8 | static_cast<uint64_t>(255 - digit);
    __syncthreads();
  }
  return gather(row, scale, s, values, values, shift, prefix);
}

// Largest and lowest value of a row (its part); +infinity for NaN too, which no
// row is sampled with.
template <int kThreads, typename T>
__device__ inline float2 row_range(const Row<T> &row, float *scratch) {
  float top = -INFINITY, low = INFINITY;
  bool bad = false;
  row.template each<kThreads, 4>([&](float v, int) {
    bad |= v != v;
    top = fmaxf(top, v);
    low = fminf(low, v);
  });
  top = block_reduce<kThreads>(bad ? INFINITY : top, scratch, Most{});
  low = block_reduce<kThreads>(low, scratch, Least{});
  return make_float2(top, low);
}

// Adds a row's (its part's) tokens to the histogram in LDS; weights only where
// `weighted`. Returns this thread's weight of what min-p keeps (a beginning of the
// order too, as the weight falls along it).
template <int kThreads, typename T>
__device__ inline uint64_t fill_bins(const Row<T> &row, typename Row<T>::wide (&now)[2],
                                     const Scale &scale, bool weighted, uint64_t least,
                                     uint32_t *count, uint64_t *mass, const double *powers) {
  uint64_t kept = 0;
  const auto add = [&](float v, bool keep) {
    const int bin = scale.bin(v);
    if (bin < 0)
      return;
    const uint64_t w = scale.weight(v, powers);
    atomicAdd(&count[bin], 1U);
    atomicAdd(reinterpret_cast<unsigned long long *>(&mass[bin]),
              static_cast<unsigned long long>(w));
    if (keep)
      kept += w >= least ? w : 0;
  };
  if (!weighted)
    row.template each<kThreads, 2>(now, [&](float v, int) {
      const int bin = scale.bin(v);
      if (bin >= 0)
        atomicAdd(&count[bin], 1U);
    });
  else if (least > 0)
    row.template each<kThreads, 2>(now, [&](float v, int) { add(v, true); });
  else
    row.template each<kThreads, 2>(now, [&](float v, int) { add(v, false); });
  return kept;
}

// Few rows of a large vocabulary run in three launches: ranges of a row's parts,
// their histograms, and a block per row that joins them and finds the borders.
// Histograms are integers: the split does not show in them.
constexpr int kSplitBins = 1024;
struct SplitRows {
  int parts, part;   // of a row; tokens of a part, a multiple of 8
  float2 *range;     // [rows][parts]
  uint64_t *kept;    // [rows][parts]
  uint64_t *mass;    // [rows][parts][kSplitBins]
  uint32_t *count;
  // A lane a part (there are at most 64); all lanes of a wave call it.
  __device__ float2 whole_range(size_t r) const {
    const int lane = threadIdx.x & 63;
    const float2 v = lane < parts ? range[r * parts + lane] : make_float2(-INFINITY, INFINITY);
    return make_float2(wave_reduce(v.x, Most{}), wave_reduce(v.y, Least{}));
  }
};

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void sample_range_kernel(const SampleArgs a,
                                                                const SplitRows split) {
  __shared__ float scratch[kThreads / 64];
  const size_t r = blockIdx.x / split.parts;
  const int first = static_cast<int>(blockIdx.x % split.parts) * split.part;
  const Row<T> row(a, r, first, min(split.part, a.vocab - first));
  const float2 range = row_range<kThreads>(row, scratch);
  if (threadIdx.x == 0)
    split.range[blockIdx.x] = range;
}

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs a,
                                                               const SplitRows split) {
  __shared__ uint64_t mass[kSplitBins];
  __shared__ uint32_t count[kSplitBins];
  __shared__ uint64_t scratch[kThreads / 64];
  __shared__ double powers[64];
  const size_t r = blockIdx.x / split.parts;
  const int first = static_cast<int>(blockIdx.x % split.parts) * split.part;
  const Row<T> row(a, r, first, min(split.part, a.vocab - first));
  typename Row<T>::wide now[2];
  row.template load<kThreads, 2>(now);
  const Cuts cuts(a, r);
  const float2 range = split.whole_range(r);
  if (!cuts.samples(range.x) || cuts.greedy())
    return;
  const bool weighted = !cuts.has_k(a.vocab);
  for (int i = threadIdx.x; i < kSplitBins; i += kThreads) {
    count[i] = 0;
    mass[i] = 0;
  }
  if (threadIdx.x < 64)
    powers[threadIdx.x] = kPowers[threadIdx.x] * a.units;
  __syncthreads();
  const Scale scale(a, range.x, range.y, cuts.temperature, kSplitBins);
  uint64_t kept =
      fill_bins<kThreads>(row, now, scale, weighted, cuts.least(), count, mass, powers);
  kept = block_reduce<kThreads>(kept, scratch, Sum{});
  __syncthreads();
  const size_t at = static_cast<size_t>(blockIdx.x) * kSplitBins;
  for (int i = threadIdx.x; i < kSplitBins; i += kThreads) {
    split.count[at + i] = count[i];
    if (weighted)
      split.mass[at + i] = mass[i];
  }
  if (threadIdx.x == 0)
    split.kept[blockIdx.x] = kept;
}

// A block per row. A row with top-k counts its bins first: where the tokens up to
// the k-th one's bin fit the list, everything else happens there.
template <typename T, int kThreads, int kBins, int kList, bool kSplit>
__global__ __launch_bounds__(kThreads) void sample_block_kernel(const SampleArgs a,
                                                                const SplitRows split) {
  static_assert(!kSplit || kBins == kSplitBins, "the parts' histograms");
  __shared__ SampleShared<kThreads, kBins, kList> s;
  __shared__ float scratch_f[kThreads / 64];
  __shared__ int scratch_i[kThreads / 64];
  __shared__ uint64_t scratch_u[kThreads / 64];
  const size_t r = blockIdx.x;
  const Row<T> row(a, r, 0, a.vocab);
  const Cuts cuts(a, r);
  // (With its parts' histograms at hand a row starts from their sums.)
  const auto sum_parts = [&](bool weighted) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      uint32_t c = 0;
      uint64_t m = 0;
      const size_t at = r * split.parts * kBins + i;
      for (int p0 = 0; p0 < split.parts; p0 += 8) {  // eight loads at a time
        uint32_t cs[8];
        uint64_t ms[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const bool has = p0 + p < split.parts;
          const size_t from = at + static_cast<size_t>(has ? p0 + p : 0) * kBins;
          cs[p] = has ? split.count[from] : 0;
          ms[p] = has && weighted ? split.mass[from] : 0;
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          c += cs[p];
          m += ms[p];
        }
      }
      s.count[i] = c;
      s.mass[i] = m;
    }
  };
  const auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
  };
  if (threadIdx.x < 64)
    s.powers[threadIdx.x] = kPowers[threadIdx.x] * a.units;
  const float2 range = kSplit ? split.whole_range(r) : row_range<kThreads>(row, scratch_f);
  const float top = range.x;
  if (!cuts.samples(top)) {
    if (threadIdx.x == 0)
      a.tokens[r] = kNoToken;
    return;
  }
  if (cuts.greedy()) {
    int first = a.vocab;
    row.template each<kThreads, 4>([&](float v, int i) {
      first = v == top ? min(first, i) : first;
    });
    first = block_reduce<kThreads>(first, scratch_i, Least{});
    if (threadIdx.x == 0)
      a.tokens[r] = static_cast<uint32_t>(first);
    return;
  }
  const Scale scale(a, top, range.y, cuts.temperature, kBins);
  const uint64_t least = cuts.least();
  const bool has_k = cuts.has_k(a.vocab);
  const uint32_t rank = static_cast<uint32_t>(cuts.top_k) - 1;
  uint64_t total = 0, kept = 0;
  uint32_t count = 0;  // tokens of weight, or listed
  bool listed = false;
  if (has_k) {
    if (kSplit) {
      sum_parts(false);
    } else {
      typename Row<T>::wide now[2];
      row.template load<kThreads, 2>(now);
      clear();
      __syncthreads();
      fill_bins<kThreads>(row, now, scale, false, least, s.count, s.mass, s.powers);
    }
    __syncthreads();
    const uint32_t last = s.count[kBins - 1];
    __syncthreads();
    scan_bins<kThreads>(s.count, s.mass, kBins, s.wave_count, s.wave_mass);
    const uint32_t all = s.count[kBins - 1] + last;
    // (Tokens without weight are not counted: with fewer than k, all are kept.)
    const int bin = last_at_most(s.count, kBins, min(rank, all - 1));
    count = bin == kBins - 1 ? all : s.count[bin + 1];
    if (count <= kList) {
      listed = true;
      const Values all_kept = scale.values(0, bin);
      count = gather(row, scale, s, all_kept, all_kept, 56, 0);
      for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        total += s.list_mass[i];
        kept += s.list_mass[i] >= least ? s.list_mass[i] : 0;
      }
      total = block_reduce<kThreads>(total, scratch_u, Sum{});
    }
    __syncthreads();
  }
  if (!listed) {
    if (kSplit && !has_k) {
      sum_parts(true);
      for (int p = threadIdx.x; p < split.parts; p += kThreads)
        kept += split.kept[r * split.parts + p];
    } else {
      typename Row<T>::wide now[2];
      row.template load<kThreads, 2>(now);
      clear();
      __syncthreads();
      kept = fill_bins<kThreads>(row, now, scale, true, least, s.count, s.mass, s.powers);
    }
    __syncthreads();
    const uint32_t last_count = s.count[kBins - 1];
    const uint64_t last_mass = s.mass[kBins - 1];
    __syncthreads();
    scan_bins<kThreads>(s.count, s.mass, kBins, s.wave_count, s.wave_mass);
    count = s.count[kBins - 1] + last_count;
    total = s.mass[kBins - 1] + last_mass;
  }
  if (cuts.min_p > 0.0F)
    kept = block_reduce<kThreads>(kept, scratch_u, Sum{});
  const auto in_bins = [&](int first, int last) {  // their tokens
    return (last == kBins - 1 ? count : s.count[last + 1]) - s.count[first];
  };
  const auto drawn = [&](uint64_t of) {
    return cuts.draw(cuts.min_p > 0.0F ? Least{}(of, kept) : of);
  };
  // The top-k border, the nucleus' border, the draw: one after the other through the
  // same code. The draw's bin depends on the nucleus' border only by that border's
  // place inside its own bin: the bins it may be in are listed along with that one.
  uint64_t at = 0;
  bool joint = false;
  uint32_t size = count;
#pragma unroll 1
  for (int border = 0; border < 3; ++border) {
    const bool by_count = border == 0;
    uint64_t target, before = 0;
    if (border == 0) {
      if (!has_k || rank >= count - 1)
        continue;
      target = rank;
    } else if (border == 1) {
      if (cuts.top_p >= 1.0F)
        continue;
      target = cuts.nucleus(total);
    } else {
      target = drawn(total);
    }
    uint32_t members = count;
    uint64_t last = 0, first = ~0ULL;
    if (!listed) {
      const int bin = by_count ? last_at_most(s.count, kBins, static_cast<uint32_t>(target))
                               : last_at_most(s.mass, kBins, target);
      members = in_bins(bin, bin);
      before = s.mass[bin];
      target -= by_count ? s.count[bin] : before;
      if (border == 1) {
        const uint64_t through = bin == kBins - 1 ? total : Least{}(total, s.mass[bin + 1]);
        const int low = last_at_most(s.mass, kBins, drawn(before + 1));
        const int high = last_at_most(s.mass, kBins, drawn(through));
        joint = members + in_bins(low, high) <= kList;
        if (joint) {
          size = gather(row, scale, s, scale.values(bin, bin), scale.values(low, high), 56, 0);
        }
      }
      if (joint) {
        const Values values = scale.values(bin, bin);
        last = values.last();
        first = values.first();
      } else {
        size = list_bin(row, scale, s, bin, by_count, members, target, before);
      }
    }
    at = find_in_list(s, size, last, first, members, by_count, target, &total);
    total += before;
    __syncthreads();
  }
  if (threadIdx.x == 0)
    a.tokens[r] = token_of(at);
}

// Parts of a row: several where rows are long and too few to fill the chip, enough
// for four blocks a CU, of 8192 tokens and more. us in parts and whole, BF16: 1 row of
// 32000 27 and 28, of 65536 31 and 41, of 131072 36 and 65; 64 rows of 65536 42 and 46,
// 128 rows of 65536 48 and 47, of 131072 62 and 73; 256 rows of 131072 85 and 78.
int parts_of(size_t rows, size_t vocab) {
  if (vocab < 32768 || rows > vocab / 1024)
    return 1;
  return static_cast<int>(
      std::min<size_t>({(1024 + rows - 1) / rows, (vocab + 8191) / 8192, 64}));
}
size_t split_bytes(size_t rows, size_t parts) {
  return rows * parts * (kSplitBins * (sizeof(uint64_t) + sizeof(uint32_t)) + sizeof(uint64_t) +
                         sizeof(float2));
}

template <typename T>
Status launch_sample(const SampleArgs &args, size_t rows, void *workspace, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(rows));
  const size_t vocab = static_cast<size_t>(args.vocab);
  SplitRows split{};
  split.parts = workspace == nullptr ? 1 : parts_of(rows, vocab);
  // A wave a row to 1024 values (us, with blocks of 256 threads in brackets: 1 row of
  // 1024 8.5 (11.9), 2048 rows 15 (37)), then blocks of 256 threads or 1024. us of both:
  // 256 rows of 9000 25 and 25, of 16000 32 and 29, of 32000 46 and 38; 512 rows of 16000
  // 36 and 52, of 32000 55 and 68, of 65536 95 and 102, of 131072 235 and 172.
  const bool narrow = vocab <= (rows <= 256 ? 8192 : 65536);
  if (args.vocab <= 512) {
    hipLaunchKernelGGL((sample_wave_kernel<T, 8>), grid, dim3(64), 0, stream, args);
  } else if (args.vocab <= 1024) {
    hipLaunchKernelGGL((sample_wave_kernel<T, 16>), grid, dim3(64), 0, stream, args);
  } else if (narrow) {
    hipLaunchKernelGGL((sample_block_kernel<T, 256, 1024, 512, false>), grid, dim3(256), 0,
                       stream, args, split);
  } else if (split.parts == 1) {
    hipLaunchKernelGGL((sample_block_kernel<T, 1024, 1024, 2048, false>), grid, dim3(1024), 0,
                       stream, args, split);
  } else {
    const size_t parts = static_cast<size_t>(split.parts);
    split.part = static_cast<int>(((vocab + parts - 1) / parts + 7) / 8 * 8);
    // (Rounded up, fewer parts may do.)
    split.parts = static_cast<int>((vocab + split.part - 1) / split.part);
    split.mass = static_cast<uint64_t *>(workspace);
    split.kept = split.mass + rows * parts * kSplitBins;
    split.range = reinterpret_cast<float2 *>(split.kept + rows * parts);
    split.count = reinterpret_cast<uint32_t *>(split.range + rows * parts);
    const dim3 blocks(static_cast<unsigned>(rows * split.parts));
    hipLaunchKernelGGL((sample_range_kernel<T, 512>), blocks, dim3(512), 0, stream, args, split);
    EVO_TRY(launch_status("sample_range_kernel"));
    hipLaunchKernelGGL((sample_bins_kernel<T, 512>), blocks, dim3(512), 0, stream, args, split);
    EVO_TRY(launch_status("sample_bins_kernel"));
    hipLaunchKernelGGL((sample_block_kernel<T, 1024, 1024, 2048, true>), grid, dim3(1024), 0,
                       stream, args, split);
  }
  return launch_status("sample_kernel");
}

}  // namespace

constexpr size_t kMostRows = size_t{1} << 20;  // a launch counts its threads in 32 bits

size_t sample_workspace_bytes(size_t rows, size_t vocab) {
  if (rows == 0 || rows > kMostRows || vocab == 0 || vocab > (size_t{1} << 20))
    return 0;
  const int parts = parts_of(rows, vocab);
  return parts == 1 ? 0 : split_bytes(rows, static_cast<size_t>(parts));
}

Status sample_tokens(int dtype, const void *logits, size_t rows, size_t vocab, size_t row_stride,
                     const float *temperature, const int32_t *top_k, const float *top_p,
                     const float *min_p, const float *uniform, uint32_t *tokens, void *workspace,
                     size_t workspace_bytes, hipStream_t stream) {
  if (logits == nullptr || uniform == nullptr || tokens == nullptr || rows == 0 ||
      rows > kMostRows || vocab == 0 || vocab > (size_t{1} << 20) || row_stride < vocab)
    return {ErrorCode::kInvalidArgument,
            "sample: null tensor, rows outside 1 .. 2^20, or a vocabulary outside 1 .. 2^20"};
  if (dtype != kElementF32 && dtype != kElementBF16 && dtype != kElementF16)
    return {ErrorCode::kInvalidArgument, "sample: logits are F32, BF16 or F16"};
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == kElementF32 ? 4 : 2) != 0)
    return {ErrorCode::kInvalidArgument, "sample: misaligned logits"};
  if (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
                               workspace_bytes < sample_workspace_bytes(rows, vocab)))
    return {ErrorCode::kInvalidArgument, "sample: workspace too small or not 16-byte aligned"};
  int log2_vocab = 0;  // rounded up
  while ((size_t{1} << log2_vocab) < vocab)
    ++log2_vocab;
  const int bits = std::min(51, 63 - log2_vocab);
  const SampleArgs args{logits, static_cast<int>(vocab), row_stride, temperature, top_k, top_p,
                        min_p, uniform, tokens, std::ldexp(1.0, bits),
                        0.6931471805599453 * (bits + 2)};
  if (dtype == kElementF32)
    return launch_sample<float>(args, rows, workspace, stream);
  if (dtype == kElementBF16)
    return launch_sample<__bf16>(args, rows, workspace, stream);
  return launch_sample<_Float16>(args, rows, workspace, stream);
}

}  // namespace evo::hip
