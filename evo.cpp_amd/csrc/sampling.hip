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
// series to the fifth power (the next term is below 2^-60).
__device__ inline uint64_t weight_units(double z, const double *powers) {
  const double n = __builtin_rint(z);
  const double r = (z - n) * 0.01083042469326756;  // ln(2) / 64
  double e = 1.0 / 120.0;
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
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

// A row's histogram and the tokens of one bin.
template <int kThreads, int kBins, int kList> struct SampleShared {
  uint64_t mass[kBins];   // before the scan a bin's own, then of the bins before it
  uint32_t count[kBins];
  uint64_t list_place[kList], list_mass[kList];
  uint64_t sub_mass[256];
  uint32_t sub_count[256];
  uint64_t wave_mass[kThreads / 64];
  uint32_t wave_count[kThreads / 64];
  double powers[64];
  uint64_t found_place, found_mass;
  uint32_t fill, found_bin;
};

template <typename T> struct Row {
  const T *logits;
  int vocab;
  float top, reach, bin_scale;
  double unit;  // 64 / (ln 2 * temperature)
  int bins;
  bool vector;  // the row starts on 16 bytes
  __device__ float at(int i) const { return static_cast<float>(logits[i]); }
  // f(value, index) over the tokens first .. end - 1 (first a multiple of 8),
  // 16 bytes a load and four loads ahead where the row is aligned.
  template <int kThreads, typename F> __device__ void each(int first, int end, F &&f) const {
    constexpr int kPer = 16 / sizeof(T), kAhead = 4;
    typedef T wide __attribute__((ext_vector_type(kPer)));
    int tail = first;
    if (vector) {
      const int whole = (end - first) / kPer;
      const wide *src = reinterpret_cast<const wide *>(logits + first);
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
              f(static_cast<float>(v[a][e]), first + (c0 + a * kThreads) * kPer + e);
          }
      }
      tail = first + whole * kPer;
    }
    for (int i = tail + threadIdx.x; i < end; i += kThreads)
      f(at(i), i);
  }
  // Bin of a value, -1 for one without weight. Every step is monotonic.
  __device__ int bin(float v) const {
    const float below = top - v;
    if (!(below <= reach))
      return -1;
    return static_cast<int>(fminf(below * bin_scale, static_cast<float>(bins - 1)));
  }
  __device__ uint64_t weight(float v, const double *powers) const {
    const double z = (static_cast<double>(v) - static_cast<double>(top)) * unit;
    return z < -2862.0 ? 0 : weight_units(z, powers);
  }
};

// Exclusive scan of count and mass over `size` entries (a multiple of the
// threads or fewer than them); returns the totals.
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
    const uint32_t bc = __shfl_up(c, offset, 64);
    const uint64_t bm = __shfl_up(m, offset, 64);
    if (lane >= offset) {
      c += bc;
      m += bm;
    }
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

// The first token, in order, of bin `bin` at which the running count (by_count)
// or weight of the bin's tokens passes `target`: its place, and the weight up to
// it, itself included. `members`: the bin's tokens.
template <typename T, int kThreads, int kBins, int kList>
__device__ inline void find_in_bin(const Row<T> &row, SampleShared<kThreads, kBins, kList> &s,
                                   int bin, uint32_t members, bool by_count, uint64_t target,
                                   uint64_t *at, uint64_t *mass) {
  // Tokens whose place begins with `prefix` in its bits above `shift`; mass before.
  uint64_t prefix = 0, before = 0;
  int shift = 56;
  while (members > kList) {
    // More than the list holds (many equal logits): 8 bits of the place at a time.
    shift -= 8;
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.sub_count[i] = 0;
      s.sub_mass[i] = 0;
    }
    __syncthreads();
    row.template each<kThreads>(0, row.vocab, [&](float v, int i) {
      if (row.bin(v) != bin)
        return;
      const uint64_t p = place(v, i);
      if (p >> (shift + 8) != prefix)
        return;
      const int digit = 255 - static_cast<int>((p >> shift) & 255);  // earlier first
      atomicAdd(&s.sub_count[digit], 1U);
      atomicAdd(reinterpret_cast<unsigned long long *>(&s.sub_mass[digit]),
                static_cast<unsigned long long>(row.weight(v, s.powers)));
    });
    __syncthreads();
    scan_bins<kThreads>(s.sub_count, s.sub_mass, 256, s.wave_count, s.wave_mass);
    // Equal entries: the last of them is the one with tokens behind it.
    const int digit = by_count
                          ? last_at_most(s.sub_count, 256, static_cast<uint32_t>(target))
                          : last_at_most(s.sub_mass, 256, target);
    const uint32_t first = s.sub_count[digit];
    members = (digit == 255 ? members : s.sub_count[digit + 1]) - first;
    before += s.sub_mass[digit];
    target -= by_count ? first : s.sub_mass[digit];
    prefix = prefix << 8 | static_cast<uint64_t>(255 - digit);
    __syncthreads();
  }
  if (threadIdx.x == 0)
    s.fill = 0;
  __syncthreads();
  row.template each<kThreads>(0, row.vocab, [&](float v, int i) {
    if (row.bin(v) != bin)
      return;
    const uint64_t p = place(v, i);
    if (p >> shift != prefix)
      return;
    const uint32_t slot = atomicAdd(&s.fill, 1U);
    s.list_place[slot] = p;
    s.list_mass[slot] = row.weight(v, s.powers);
  });
  __syncthreads();
  // Rank by comparison: the one token whose range holds the target.
  const uint32_t size = s.fill;
  for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
    const uint64_t p = s.list_place[i];
    uint64_t ahead = 0;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < size; ++j)
      if (s.list_place[j] > p) {
        ahead += s.list_mass[j];
        ++rank;
      }
    const uint64_t own = s.list_mass[i];
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

template <typename T, int kThreads, int kBins, int kList>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a) {
  __shared__ SampleShared<kThreads, kBins, kList> s;
  __shared__ float scratch_f[kThreads / 64];
  __shared__ int scratch_i[kThreads / 64];
  __shared__ uint64_t scratch_u[kThreads / 64];
  const size_t r = blockIdx.x;
  Row<T> row;
  row.logits = static_cast<const T *>(a.logits) + r * a.row_stride;
  row.vocab = a.vocab;
  row.vector = reinterpret_cast<uintptr_t>(row.logits) % 16 == 0;
  row.bins = kBins;
  const float temperature = a.temperature == nullptr ? 1.0F : a.temperature[r];
  const int top_k = a.top_k == nullptr ? 0 : a.top_k[r];
  const float top_p = a.top_p == nullptr ? 1.0F : a.top_p[r];
  const float min_p = a.min_p == nullptr ? 0.0F : a.min_p[r];
  const float uniform = a.uniform[r];

  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  if (threadIdx.x < 64)
    s.powers[threadIdx.x] = kPowers[threadIdx.x];

  float top = -INFINITY, low = INFINITY;
  int bad = 0;
  row.template each<kThreads>(0, a.vocab, [&](float v, int) {
    bad |= !(v < INFINITY);
    top = fmaxf(top, v);
    low = v > -INFINITY ? fminf(low, v) : low;
  });
  const auto most = [](float x, float y) { return fmaxf(x, y); };
  const auto least = [](float x, float y) { return fminf(x, y); };
  top = block_reduce<kThreads>(top, scratch_f, most);
  low = block_reduce<kThreads>(low, scratch_f, least);
  bad = block_reduce<kThreads>(bad, scratch_i, [](int x, int y) { return x | y; });
  if (bad != 0 || top == -INFINITY || !(temperature >= 0.0F) || !(temperature < INFINITY) ||
      top_k < 0 || !(top_p > 0.0F && top_p <= 1.0F) || !(min_p >= 0.0F && min_p <= 1.0F) ||
      uniform != uniform) {
    if (threadIdx.x == 0)
      a.tokens[r] = kNoToken;
    return;
  }
  if (temperature == 0.0F || top_k == 1) {
    int first = a.vocab;
    row.template each<kThreads>(0, a.vocab, [&](float v, int i) {
      if (v == top)
        first = min(first, i);
    });
    first = block_reduce<kThreads>(first, scratch_i, [](int x, int y) { return min(x, y); });
    if (threadIdx.x == 0)
      a.tokens[r] = static_cast<uint32_t>(first);
    return;
  }
  row.top = top;
  row.reach = static_cast<float>(fmin(kReach * static_cast<double>(temperature), 3.0e38));
  row.unit = 92.33248261893106 / static_cast<double>(temperature);  // 64 / ln(2)
  const float range = fminf(row.reach, top - low);
  row.bin_scale = range > 0.0F ? fminf(kBins / range, 3.0e38F) : 0.0F;

  // Counts and weights by bin, and the weight of what min-p keeps (a beginning
  // of the order too, as the weight falls along it).
  const double least_weight = static_cast<double>(min_p) * 4398046511104.0;
  uint64_t kept = 0;
  row.template each<kThreads>(0, a.vocab, [&](float v, int) {
    const int bin = row.bin(v);
    if (bin < 0)
      return;
    const uint64_t w = row.weight(v, s.powers);
    atomicAdd(&s.count[bin], 1U);
    atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[bin]),
              static_cast<unsigned long long>(w));
    kept += static_cast<double>(w) >= least_weight ? w : 0;
  });
  kept = block_reduce<kThreads>(kept, scratch_u, [](uint64_t x, uint64_t y) { return x + y; });
  __syncthreads();
  uint32_t total_count = 0;
  uint64_t total = 0;
  {
    const uint32_t last_count = s.count[kBins - 1];
    const uint64_t last_mass = s.mass[kBins - 1];
    __syncthreads();
    scan_bins<kThreads>(s.count, s.mass, kBins, s.wave_count, s.wave_mass);
    total_count = s.count[kBins - 1] + last_count;
    total = s.mass[kBins - 1] + last_mass;
  }
  const auto members = [&](int bin) {
    return (bin == kBins - 1 ? total_count : s.count[bin + 1]) - s.count[bin];
  };
  uint64_t at = 0, mass = 0;
  if (top_k > 0 && static_cast<uint32_t>(top_k) < total_count) {
    const uint32_t rank = static_cast<uint32_t>(top_k) - 1;
    const int bin = last_at_most(s.count, kBins, rank);
    find_in_bin(row, s, bin, members(bin), true, rank - s.count[bin], &at, &mass);
    total = s.mass[bin] + mass;
  }
  if (top_p < 1.0F) {
    // Tokens are kept while the weight before them is below top_p * total: up
    // to the first whose weight, itself included, reaches it.
    const uint64_t reach = static_cast<uint64_t>(
        __builtin_ceil(static_cast<double>(top_p) * static_cast<double>(total)));
    const uint64_t target = min(reach, total) - 1;
    const int bin = last_at_most(s.mass, kBins, target);
    find_in_bin(row, s, bin, members(bin), false, target - s.mass[bin], &at, &mass);
    total = s.mass[bin] + mass;
  }
  total = min(total, kept);
  const double drawn = fmax(static_cast<double>(uniform), 0.0) * static_cast<double>(total);
  const uint64_t target =
      drawn >= static_cast<double>(total) ? total - 1
                                          : min(static_cast<uint64_t>(drawn), total - 1);
  const int bin = last_at_most(s.mass, kBins, target);
  find_in_bin(row, s, bin, members(bin), false, target - s.mass[bin], &at, &mass);
  if (threadIdx.x == 0)
    a.tokens[r] = 0xffffffU - static_cast<uint32_t>(at & 0xffffff);
}

template <typename T>
void launch_sample(const SampleArgs &args, size_t rows, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(rows));
  if (args.vocab <= 1024)
    hipLaunchKernelGGL((sample_kernel<T, 64, 512, 256>), grid, dim3(64), 0, stream, args);
  else if (args.vocab <= 16384)
    hipLaunchKernelGGL((sample_kernel<T, 256, 1024, 512>), grid, dim3(256), 0, stream, args);
  else
    hipLaunchKernelGGL((sample_kernel<T, 1024, 2048, 1024>), grid, dim3(1024), 0, stream, args);
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
