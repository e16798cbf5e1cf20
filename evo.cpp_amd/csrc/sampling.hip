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
// integers of 2^-42: such a sum has no order, so neither the atomics of the
// histogram nor a split of a row can change a token, and a border is off by less
// than 1e-11 of the row's largest weight. A weight below 2^-43 (30 below the top,
// in units of the temperature) counts as none.
#include "common.hpp"
#include "ops.hpp"

#include <cmath>

namespace evo::hip {

namespace {

constexpr double kReach = 31.0;  // exp(-31) < 2^-43
constexpr uint32_t kNoToken = 0xffffffffU;

struct SampleArgs {
  const void *logits;
  int vocab;
  size_t row_stride;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p, *uniform;
  uint32_t *tokens;
};

// Order of the values as integers; -0 and 0 are one value.
__device__ inline uint32_t ordered(float v) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0F);
  return (bits & 0x80000000U) != 0 ? ~bits : bits | 0x80000000U;
}
// Place of a token in the order: larger is earlier. 56 bits, vocab <= 2^20.
__device__ inline uint64_t place(float v, int index) {
  return static_cast<uint64_t>(ordered(v)) << 24 | static_cast<uint32_t>(0xffffff - index);
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

// exp(x) in units of 2^-42, rounded, for x = z * ln(2) / 64 in [-32, 0]: with
// z = n + f, 2^(n / 64) from a table and a shift, exp(f ln(2) / 64) by its
// series to the fifth power in f (the next term is below 2^-60).
__device__ inline uint64_t weight_units(double z, const double *powers) {
  const double n = __builtin_rint(z), f = z - n;
  double e = 1.2417843701716925e-12;
  e = fma(e, f, 5.7328516886404019e-10);
  e = fma(e, f, 2.1173137155464776e-07);
  e = fma(e, f, 5.86490495505617e-05);
  e = fma(e, f, 0.010830424696249145);
  e = fma(e, f, 1.0);
  const int whole = static_cast<int>(n);
  const uint64_t bits = __builtin_bit_cast(uint64_t, e * powers[whole & 63]) +
                        (static_cast<uint64_t>(static_cast<int64_t>((whole >> 6) + 42)) << 52);
  // Adding 2^52 rounds to a whole number in the low bits.
  const double shifted = __builtin_bit_cast(double, bits) + 4503599627370496.0;
  return __builtin_bit_cast(uint64_t, shifted) & 0xfffffffffffffULL;
}

template <typename V, typename F> __device__ inline V wave_reduce(V v, F &&f) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1)
    v = f(v, __shfl_xor(v, offset, 64));
  return v;
}
template <int kThreads, typename V, typename F>
__device__ inline V block_reduce(V v, V *scratch, F &&f) {
  v = wave_reduce(v, f);
  if constexpr (kThreads > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
      scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < kThreads / 64; ++w)
      v = f(v, scratch[w]);
  }
  return v;
}
struct Most {
  template <typename V> __device__ V operator()(V x, V y) const { return x > y ? x : y; }
};
struct Least {
  template <typename V> __device__ V operator()(V x, V y) const { return x < y ? x : y; }
};
struct Sum {
  template <typename V> __device__ V operator()(V x, V y) const { return x + y; }
};

// A row's parameters.
struct Cuts {
  float temperature, top_p, min_p, uniform;
  int top_k;
  __device__ Cuts(const SampleArgs &a, size_t r)
      : temperature(a.temperature == nullptr ? 1.0F : a.temperature[r]),
        top_p(a.top_p == nullptr ? 1.0F : a.top_p[r]),
        min_p(a.min_p == nullptr ? 0.0F : a.min_p[r]), uniform(a.uniform[r]),
        top_k(a.top_k == nullptr ? 0 : a.top_k[r]) {}
  __device__ bool valid() const {
    return temperature >= 0.0F && temperature < INFINITY && top_k >= 0 && top_p > 0.0F &&
           top_p <= 1.0F && min_p >= 0.0F && min_p <= 1.0F && uniform == uniform;
  }
  __device__ bool greedy() const { return temperature == 0.0F || top_k == 1; }
  // Least weight that min-p keeps.
  __device__ uint64_t least() const {
    return static_cast<uint64_t>(__builtin_ceil(static_cast<double>(min_p) * 4398046511104.0));
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

// How a row's values map to bins and weights, given its largest and lowest value.
struct Scale {
  float top, reach, bin_scale;
  double unit;  // 64 / (ln 2 * temperature)
  __device__ Scale(float top_, float low, float temperature, int bins)
      : top(top_), reach(static_cast<float>(
                       fmin(kReach * static_cast<double>(temperature), 3.0e38))),
        unit(92.33248261893106 / static_cast<double>(temperature)) {
    const float range = fminf(reach, top - low);
    // A little less than bins / range: the last value stays inside.
    bin_scale = range > 0.0F ? fminf(static_cast<float>(bins) * 0.999999F / range, 3.0e38F) : 0.0F;
  }
  // Bin of a value, -1 for one without weight. Every step is monotonic.
  __device__ int bin(float v) const {
    const float below = top - v;
    return below <= reach ? static_cast<int>(below * bin_scale) : -1;
  }
  __device__ bool in_bin(float v, float first) const {  // bin(v) == first
    const float at = (top - v) * bin_scale;
    return at >= first && at < first + 1.0F && top - v <= reach;
  }
  __device__ uint64_t weight(float v, const double *powers) const {
    const double z = (static_cast<double>(v) - static_cast<double>(top)) * unit;
    return z < -2862.0 ? 0 : weight_units(z, powers);
  }
};

// ------------------------------------------------------- small vocabularies
// A wave per row, kPer values a lane in registers. A border's bin is found in the
// scanned histogram that the lanes hold, four bins each; a bin of more than a few
// tokens is histogrammed again over the range of its places; the last few are taken
// one by one.
template <typename T, int kPer>
__global__ __launch_bounds__(64) void sample_wave_kernel(const SampleArgs a) {
  constexpr int kBins = 256;
  __shared__ __attribute__((aligned(16))) uint64_t mass_s[kBins];
  __shared__ __attribute__((aligned(16))) uint32_t count_s[kBins];
  __shared__ double powers[64];
  const int lane = threadIdx.x;
  const size_t r = blockIdx.x;
  const T *logits = static_cast<const T *>(a.logits) + r * a.row_stride;
  float v[kPer];  // value e of the lane is token 64 * e + lane
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    v[e] = 64 * e + lane < a.vocab ? static_cast<float>(logits[64 * e + lane]) : -INFINITY;
  const Cuts cuts(a, r);
  powers[lane] = kPowers[lane];
  auto clear = [&] {
    reinterpret_cast<uint4 *>(mass_s)[2 * lane] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(mass_s)[2 * lane + 1] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(count_s)[lane] = make_uint4(0, 0, 0, 0);
  };
  clear();
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
  if (__any(bad) || top == -INFINITY || !cuts.valid()) {
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
  const Scale scale(top, low, cuts.temperature, kBins);
  __syncthreads();
  uint64_t w[kPer];
  int bin[kPer];
  const uint64_t least = cuts.least();
  uint64_t kept = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    bin[e] = scale.bin(v[e]);
    w[e] = bin[e] >= 0 ? scale.weight(v[e], powers) : 0;
    kept += w[e] >= least ? w[e] : 0;
    if (bin[e] >= 0) {
      atomicAdd(&count_s[bin[e]], 1U);
      atomicAdd(reinterpret_cast<unsigned long long *>(&mass_s[bin[e]]),
                static_cast<unsigned long long>(w[e]));
    }
  }
  // The lane's four bins, and what lies before them.
  struct Bins {
    uint64_t mass[4], mass_before, mass_total;
    uint32_t count[4], count_before, count_total;
  };
  auto scanned = [&] {
    Bins b;
    __syncthreads();
    uint64_t m = 0;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b.mass[j] = mass_s[4 * lane + j];
      b.count[j] = count_s[4 * lane + j];
      m += b.mass[j];
      c += b.count[j];
    }
    const uint64_t own_m = m;
    const uint32_t own_c = c;
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
      const uint64_t up_m = __shfl_up(m, offset, 64);
      const uint32_t up_c = __shfl_up(c, offset, 64);
      m += lane >= offset ? up_m : 0;
      c += lane >= offset ? up_c : 0;
    }
    b.mass_before = m - own_m;
    b.count_before = c - own_c;
    b.mass_total = __shfl(m, 63, 64);
    b.count_total = __shfl(c, 63, 64);
    __syncthreads();
    return b;
  };
  // The bin in which the running count or weight passes the target, what lies before
  // it, and how many tokens it has.
  struct Hit {
    int bin;
    uint64_t mass_before;
    uint32_t count_before, members;
  };
  auto locate = [&](const Bins &b, bool by_count, uint64_t target) {
    uint64_t at_m = b.mass_before;
    uint32_t at_c = b.count_before;
    Hit h{-1, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t from = by_count ? at_c : at_m;
      const uint64_t size = by_count ? b.count[j] : b.mass[j];
      if (target >= from && target - from < size)
        h = {4 * lane + j, at_m, at_c, b.count[j]};
      at_m += b.mass[j];
      at_c += b.count[j];
    }
    const uint64_t owner = __ballot(h.bin >= 0);
    const int from = owner == 0 ? 0 : __builtin_ctzll(owner);
    return Hit{__shfl(h.bin, from, 64), __shfl(h.mass_before, from, 64),
               static_cast<uint32_t>(__shfl(h.count_before, from, 64)),
               static_cast<uint32_t>(__shfl(h.members, from, 64))};
  };
  const Bins all = scanned();
  // The token at which the running count or weight of the order passes the target,
  // and the weight up to it, itself included.
  auto find = [&](bool by_count, uint64_t target, uint64_t *mass) {
    Hit h = locate(all, by_count, target);
    uint64_t before = h.mass_before;
    target -= by_count ? h.count_before : h.mass_before;
    uint64_t spot[kPer];  // the candidates' places, else 0
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      spot[e] = bin[e] == h.bin ? place(v[e], 64 * e + lane) : 0;
    uint32_t members = h.members;
    while (members > 6) {
      uint64_t last = ~0ULL, first = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        first = first > spot[e] ? first : spot[e];
        last = spot[e] != 0 && spot[e] < last ? spot[e] : last;
      }
      first = wave_reduce(first, Most{});
      last = wave_reduce(last, Least{});
      const int shift = max(0, 56 - static_cast<int>(__builtin_clzll(first - last)));
      clear();
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (spot[e] != 0) {
          const int sub = static_cast<int>((first - spot[e]) >> shift);
          atomicAdd(&count_s[sub], 1U);
          atomicAdd(reinterpret_cast<unsigned long long *>(&mass_s[sub]),
                    static_cast<unsigned long long>(w[e]));
        }
      h = locate(scanned(), by_count, target);
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
      own = __shfl(own, __builtin_ctzll(__ballot(first == token)), 64);
      before += own;
      if (by_count ? target == i : target < own)
        break;
      target -= by_count ? 0 : own;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        spot[e] = spot[e] == token ? 0 : spot[e];
    }
    *mass = before;
    return 0xffffffU - static_cast<uint32_t>(token & 0xffffff);
  };
  uint64_t total = all.mass_total;
  if (cuts.top_k > 0 && static_cast<uint32_t>(cuts.top_k) < all.count_total)
    find(true, static_cast<uint64_t>(cuts.top_k) - 1, &total);
  if (cuts.top_p < 1.0F)
    find(false, cuts.nucleus(total), &total);
  if (cuts.min_p > 0.0F) {
    kept = wave_reduce(kept, Sum{});
    total = total < kept ? total : kept;
  }
  uint64_t through;
  const uint32_t token = find(false, cuts.draw(total), &through);
  if (lane == 0)
    a.tokens[r] = token;
}

// ------------------------------------------------------- large vocabularies
template <typename T> struct Row {
  const T *logits;
  int vocab;
  bool vector;  // the row starts on 16 bytes
  // f(value, index) over the tokens, 16 bytes a load and four loads ahead where the
  // row is aligned.
  template <int kThreads, typename F> __device__ void each(F &&f) const {
    constexpr int kPer = 16 / sizeof(T), kAhead = 4;
    typedef T wide __attribute__((ext_vector_type(kPer)));
    int tail = 0;
    if (vector) {
      const int whole = vocab / kPer;
      const wide *src = reinterpret_cast<const wide *>(logits);
      for (int c0 = threadIdx.x; c0 < whole; c0 += kThreads * kAhead) {
        wide v[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (c0 + a * kThreads < whole)
            v[a] = src[c0 + a * kThreads];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (c0 + a * kThreads < whole) {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
              f(static_cast<float>(v[a][e]), (c0 + a * kThreads) * kPer + e);
          }
      }
      tail = whole * kPer;
    }
    for (int i = tail + threadIdx.x; i < vocab; i += kThreads)
      f(static_cast<float>(logits[i]), i);
  }
};

// A row's histogram and a list of tokens.
template <int kThreads, int kBins, int kList> struct SampleShared {
  uint64_t mass[kBins];   // before the scan a bin's own, then of the bins before it
  uint32_t count[kBins];
  uint64_t list_place[kList], list_mass[kList];
  uint64_t sub_mass[256], few_place[64], few_mass[64];
  uint32_t sub_count[256];
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
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const uint32_t up_c = __shfl_up(c, offset, 64);
    const uint64_t up_m = __shfl_up(m, offset, 64);
    c += lane >= offset ? up_c : 0;
    m += lane >= offset ? up_m : 0;
  }
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

// The listed token, in order, at which the running count (by_count) or weight of the
// list's `members` passes the target: its place, and the weight up to it, itself
// included. More than 64 are narrowed by histograms over the range of their places.
template <int kThreads, int kBins, int kList>
__device__ inline void find_in_list(SampleShared<kThreads, kBins, kList> &s, uint32_t members,
                                    bool by_count, uint64_t target, uint64_t *at,
                                    uint64_t *mass) {
  __shared__ uint64_t scratch[kThreads / 64];
  const uint32_t size = members;
  uint64_t last = 0, first = ~0ULL, before = 0;  // places taken into account
  while (members > 64) {
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
      if (p >= last && p <= first) {
        const int sub = static_cast<int>((hi - p) >> shift);
        atomicAdd(&s.sub_count[sub], 1U);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.sub_mass[sub]),
                  static_cast<unsigned long long>(s.list_mass[i]));
      }
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
      s.few_place[slot] = p;
      s.few_mass[slot] = s.list_mass[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < members) {
    const uint64_t p = s.few_place[threadIdx.x], own = s.few_mass[threadIdx.x];
    uint64_t ahead = 0;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < members; ++j)
      if (s.few_place[j] > p) {
        ahead += s.few_mass[j];
        ++rank;
      }
    if (by_count ? rank == target : ahead <= target && target < ahead + own) {
      s.found_place = p;
      s.found_mass = before + ahead + own;
    }
  }
  __syncthreads();
  *at = s.found_place;
  *mass = s.found_mass;
  __syncthreads();
}

// Lists the tokens that `take` wants, and their weights.
template <typename T, int kThreads, int kBins, int kList, typename F>
__device__ inline void gather(const Row<T> &row, const Scale &scale,
                              SampleShared<kThreads, kBins, kList> &s, F &&take) {
  if (threadIdx.x == 0)
    s.fill = 0;
  __syncthreads();
  row.template each<kThreads>([&](float v, int i) {
    if (!take(v, i))
      return;
    const uint32_t slot = atomicAdd(&s.fill, 1U);
    s.list_place[slot] = place(v, i);
    s.list_mass[slot] = scale.weight(v, s.powers);
  });
  __syncthreads();
}

// find_in_list over the `members` tokens of a bin.
template <typename T, int kThreads, int kBins, int kList>
__device__ inline void find_in_bin(const Row<T> &row, const Scale &scale,
                                   SampleShared<kThreads, kBins, kList> &s, int bin,
                                   uint32_t members, bool by_count, uint64_t target,
                                   uint64_t *at, uint64_t *mass) {
  // Tokens whose place begins with `prefix` in its bits above `shift`; mass before.
  uint64_t prefix = 0, before = 0;
  int shift = 56;
  const float first_bin = static_cast<float>(bin);
  while (members > kList) {
    // More than the list holds (many equal logits): 8 bits of the place at a time.
    shift -= 8;
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.sub_count[i] = 0;
      s.sub_mass[i] = 0;
    }
    __syncthreads();
    row.template each<kThreads>([&](float v, int i) {
      if (!scale.in_bin(v, first_bin))
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
  gather(row, scale, s, [&](float v, int i) {
    return scale.in_bin(v, first_bin) && place(v, i) >> shift == prefix;
  });
  find_in_list(s, members, by_count, target, at, mass);
  *mass += before;
}

// A block per row. A row with top-k counts its bins first: where the tokens up to
// the k-th one's bin fit the list, everything else happens there.
template <typename T, int kThreads, int kBins, int kList>
__global__ __launch_bounds__(kThreads) void sample_block_kernel(const SampleArgs a) {
  __shared__ SampleShared<kThreads, kBins, kList> s;
  __shared__ float scratch_f[kThreads / 64];
  __shared__ int scratch_i[kThreads / 64];
  __shared__ uint64_t scratch_u[kThreads / 64];
  const size_t r = blockIdx.x;
  Row<T> row;
  row.logits = static_cast<const T *>(a.logits) + r * a.row_stride;
  row.vocab = a.vocab;
  row.vector = reinterpret_cast<uintptr_t>(row.logits) % 16 == 0;
  const Cuts cuts(a, r);
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  if (threadIdx.x < 64)
    s.powers[threadIdx.x] = kPowers[threadIdx.x];

  float top = -INFINITY, low = INFINITY;
  bool bad = false;
  row.template each<kThreads>([&](float v, int) {
    bad |= v != v;
    top = fmaxf(top, v);
    low = fminf(low, v);
  });
  top = block_reduce<kThreads>(top, scratch_f, Most{});
  low = block_reduce<kThreads>(low, scratch_f, Least{});
  if (__syncthreads_or(bad) || !(top < INFINITY) || top == -INFINITY || !cuts.valid()) {
    if (threadIdx.x == 0)
      a.tokens[r] = kNoToken;
    return;
  }
  if (cuts.greedy()) {
    int first = a.vocab;
    row.template each<kThreads>([&](float v, int i) {
      first = v == top ? min(first, i) : first;
    });
    first = block_reduce<kThreads>(first, scratch_i, Least{});
    if (threadIdx.x == 0)
      a.tokens[r] = static_cast<uint32_t>(first);
    return;
  }
  const Scale scale(top, low, cuts.temperature, kBins);
  const uint64_t least = cuts.least();
  const bool has_k = cuts.top_k > 0 && cuts.top_k < a.vocab;
  const uint32_t rank = static_cast<uint32_t>(cuts.top_k) - 1;
  uint64_t at = 0, mass = 0, total = 0, kept = 0;
  if (has_k) {
    row.template each<kThreads>([&](float v, int) {
      const int bin = scale.bin(v);
      if (bin >= 0)
        atomicAdd(&s.count[bin], 1U);
    });
    __syncthreads();
    const uint32_t last = s.count[kBins - 1];
    __syncthreads();
    scan_bins<kThreads>(s.count, s.mass, kBins, s.wave_count, s.wave_mass);
    const uint32_t all = s.count[kBins - 1] + last;
    // (Tokens without weight are not counted: with fewer than k, all are kept.)
    const int bin = last_at_most(s.count, kBins, min(rank, all - 1));
    const uint32_t through = bin == kBins - 1 ? all : s.count[bin + 1];
    if (through <= kList) {
      const float end = static_cast<float>(bin + 1);
      gather(row, scale, s, [&](float v, int) {
        return (top - v) * scale.bin_scale < end && top - v <= scale.reach;
      });
      if (rank < all - 1) {
        find_in_list(s, through, true, rank, &at, &total);
      } else {
        uint64_t sum = 0;
        for (uint32_t i = threadIdx.x; i < through; i += kThreads)
          sum += s.list_mass[i];
        total = block_reduce<kThreads>(sum, scratch_u, Sum{});
      }
      if (cuts.top_p < 1.0F)
        find_in_list(s, through, false, cuts.nucleus(total), &at, &total);
      if (cuts.min_p > 0.0F) {
        for (uint32_t i = threadIdx.x; i < through; i += kThreads)
          kept += s.list_mass[i] >= least ? s.list_mass[i] : 0;
        kept = block_reduce<kThreads>(kept, scratch_u, Sum{});
        total = Least{}(total, kept);
      }
      find_in_list(s, through, false, cuts.draw(total), &at, &mass);
      if (threadIdx.x == 0)
        a.tokens[r] = 0xffffffU - static_cast<uint32_t>(at & 0xffffff);
      return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
  }
  // Counts and weights by bin, and the weight of what min-p keeps (a beginning of the
  // order too, as the weight falls along it).
  row.template each<kThreads>([&](float v, int) {
    const int bin = scale.bin(v);
    if (bin < 0)
      return;
    const uint64_t w = scale.weight(v, s.powers);
    atomicAdd(&s.count[bin], 1U);
    atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[bin]),
              static_cast<unsigned long long>(w));
    if (least > 0)
      kept += w >= least ? w : 0;
  });
  __syncthreads();
  const uint32_t last_count = s.count[kBins - 1];
  const uint64_t last_mass = s.mass[kBins - 1];
  __syncthreads();
  scan_bins<kThreads>(s.count, s.mass, kBins, s.wave_count, s.wave_mass);
  const uint32_t total_count = s.count[kBins - 1] + last_count;
  total = s.mass[kBins - 1] + last_mass;
  const auto members = [&](int bin) {
    return (bin == kBins - 1 ? total_count : s.count[bin + 1]) - s.count[bin];
  };
  if (has_k && rank < total_count - 1) {
    const int bin = last_at_most(s.count, kBins, rank);
    find_in_bin(row, scale, s, bin, members(bin), true, rank - s.count[bin], &at, &mass);
    total = s.mass[bin] + mass;
  }
  if (cuts.top_p < 1.0F) {
    const uint64_t target = cuts.nucleus(total);
    const int bin = last_at_most(s.mass, kBins, target);
    find_in_bin(row, scale, s, bin, members(bin), false, target - s.mass[bin], &at, &mass);
    total = s.mass[bin] + mass;
  }
  if (cuts.min_p > 0.0F)
    total = Least{}(total, block_reduce<kThreads>(kept, scratch_u, Sum{}));
  const uint64_t target = cuts.draw(total);
  const int bin = last_at_most(s.mass, kBins, target);
  find_in_bin(row, scale, s, bin, members(bin), false, target - s.mass[bin], &at, &mass);
  if (threadIdx.x == 0)
    a.tokens[r] = 0xffffffU - static_cast<uint32_t>(at & 0xffffff);
}

template <typename T>
void launch_sample(const SampleArgs &args, size_t rows, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(rows));
  if (args.vocab <= 512)
    hipLaunchKernelGGL((sample_wave_kernel<T, 8>), grid, dim3(64), 0, stream, args);
  else if (args.vocab <= 1024)
    hipLaunchKernelGGL((sample_wave_kernel<T, 16>), grid, dim3(64), 0, stream, args);
  else if (args.vocab <= 16384)
    hipLaunchKernelGGL((sample_block_kernel<T, 256, 1024, 512>), grid, dim3(256), 0, stream, args);
  else
    hipLaunchKernelGGL((sample_block_kernel<T, 1024, 2048, 2048>), grid, dim3(1024), 0, stream,
                       args);
}

}  // namespace

size_t sample_workspace_bytes(size_t, size_t) { return 0; }

Status sample_tokens(int dtype, const void *logits, size_t rows, size_t vocab, size_t row_stride,
                     const float *temperature, const int32_t *top_k, const float *top_p,
                     const float *min_p, const float *uniform, uint32_t *tokens, void *workspace,
                     size_t workspace_bytes, hipStream_t stream) {
  if (logits == nullptr || uniform == nullptr || tokens == nullptr || rows == 0 ||
      rows > (size_t{1} << 30) || vocab == 0 || vocab > (size_t{1} << 20) || row_stride < vocab)
    return {ErrorCode::kInvalidArgument,
            "sample: null tensor, no rows, or a vocabulary of none or more than 2^20"};
  if (dtype != kElementF32 && dtype != kElementBF16 && dtype != kElementF16)
    return {ErrorCode::kInvalidArgument, "sample: logits are F32, BF16 or F16"};
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == kElementF32 ? 4 : 2) != 0)
    return {ErrorCode::kInvalidArgument, "sample: misaligned logits"};
  const SampleArgs args{logits, static_cast<int>(vocab), row_stride, temperature, top_k,
                        top_p, min_p, uniform, tokens};
  if (dtype == kElementF32)
    launch_sample<float>(args, rows, stream);
  else if (dtype == kElementBF16)
    launch_sample<__bf16>(args, rows, stream);
  else
    launch_sample<_Float16>(args, rows, stream);
  return launch_status("sample_kernel");
}

}  // namespace evo::hip
