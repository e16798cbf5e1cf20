// SPDX-License-Identifier: Apache-2.0
// Low-rank adapters of many requests beside a shared product:
//   out[t] = residual[t] + s_a U_a (D_a x[t]),  a the adapter of row t (or none).
//
// Rows are sorted by adapter on the device (group_kernel), so that an adapter is read
// once for up to 64 of its rows wherever they lie. down_kernel forms the inner values
// D_a x of such a tile for a part of the width, up_kernel adds the parts up, scales them
// and forms a chunk of the output columns. Both take their operands from memory to
// registers: a 16 x 16 x 32 matrix instruction wants 16 bytes of a row from each lane.
// x comes as the planes hi (+ lo) of a split-BF16 activation, whose products with BF16
// weights are exact in F32. The inner values are F32, and stay so in the second product:
// each is cut into three BF16 planes, 8 bits each, which hold all of its 24.
// A row's values come from its own column of each product: an infinity or NaN of one row
// or adapter reaches no other row.
#include "common.hpp"
#include "lanes.hpp"
#include "ops.hpp"

#include <algorithm>
#include <type_traits>

namespace evo::hip {

namespace {

constexpr int kTileRows = 64, kGroupThreads = 1024;
constexpr size_t kDirectRows = 16;  // rows up to this are not sorted

struct Tile {
  int adapter, first, count;  // rows order[first ..]; adapter -1: rows without one
};

struct AdapterArgs {
  AdapterPool pool;
  const int32_t *adapter;
  const uint16_t *hi, *lo;
  size_t x_stride;
  int rows;
  const float *residual;
  float *out;
  size_t out_stride;
  int tiles;    // at most
  int parts;    // of the width, in down_kernel
  int chunk;    // output columns of a block, in up_kernel
  int direct;   // a tile is a row
  int32_t *bin;    // [rows], the adapter of each as it was read; the pool's size: none
  int32_t *order;  // [rows], sorted by it
  Tile *tile;      // [tiles], count 0 behind the last
  float *inner;    // [parts][rows][rank]
};

__device__ inline int rank_of(const AdapterPool &pool, int adapter) {
  return pool.ranks == nullptr ? pool.rank : max(0, min(pool.ranks[adapter], pool.rank));
}
// The adapter of a row; the pool's size stands for none, and for one it does not have.
__device__ inline int checked_adapter(const AdapterArgs &a, int row) {
  const int adapter = a.adapter[row];
  if (adapter == -1)
    return a.pool.adapters;
  if (adapter >= 0 && adapter < a.pool.adapters &&
      (a.pool.ranks == nullptr || a.pool.ranks[adapter] == rank_of(a.pool, adapter)))
    return adapter;
  if (a.pool.error != nullptr)
    atomicOr(a.pool.error, kBadAdapter);
  return a.pool.adapters;
}

// ------------------------------------------------------------ rows by adapter
// One block sorts the rows by counting: bin a holds the rows of adapter a, the last one
// those without.
__global__ __launch_bounds__(kGroupThreads) void group_kernel(const AdapterArgs a) {
  extern __shared__ int32_t bins[];
  __shared__ int32_t rows_before[kGroupThreads / 64], tiles_before[kGroupThreads / 64];
  const int count = a.pool.adapters + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < count; i += kGroupThreads)
    bins[i] = 0;
  __syncthreads();
  // A wave's place in a bin: one addition where all of its rows share one, as in prompts.
  const auto add = [&](int row, bool place) {
    const bool mine = row < a.rows;
    int bin = -1;
    if (mine && place)
      bin = a.bin[row];  // (which this thread wrote: both passes see one adapter)
    else if (mine)
      a.bin[row] = bin = checked_adapter(a, row);
    const int first = __builtin_amdgcn_readfirstlane(bin);
    const uint64_t same = __ballot(bin == first);
    if (__ballot(mine) == same && first >= 0) {
      int at = 0;
      if (lane == 0)
        at = atomicAdd(&bins[first], static_cast<int>(__popcll(same)));
      at = __builtin_amdgcn_readfirstlane(at);
      if (place && mine)
        a.order[at + lane] = row;
    } else if (mine) {
      const int at = atomicAdd(&bins[bin], 1);
      if (place)
        a.order[at] = row;
    }
  };
  for (int row = threadIdx.x; row < (a.rows + 63) / 64 * 64; row += kGroupThreads)
    add(row, false);
  __syncthreads();

  // Each thread's bins, and what lies before them.
  const int each = (count + kGroupThreads - 1) / kGroupThreads, from = threadIdx.x * each;
  int rows = 0, tiles = 0;
  for (int i = from; i < min(from + each, count); ++i) {
    rows += bins[i];
    tiles += (bins[i] + kTileRows - 1) / kTileRows;
  }
  int rows_through = rows, tiles_through = tiles;
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const int r = __shfl_up(rows_through, offset, 64), t = __shfl_up(tiles_through, offset, 64);
    rows_through += lane >= offset ? r : 0;
    tiles_through += lane >= offset ? t : 0;
  }
  if (lane == 63) {
    rows_before[wave] = rows_through;
    tiles_before[wave] = tiles_through;
  }
  __syncthreads();
  int at = rows_through - rows, tile = tiles_through - tiles, all = 0;
  for (int w = 0; w < kGroupThreads / 64; ++w) {
    at += w < wave ? rows_before[w] : 0;
    tile += w < wave ? tiles_before[w] : 0;
    all += tiles_before[w];
  }
  for (int i = from; i < min(from + each, count); ++i) {
    const int n = bins[i];
    bins[i] = at;
    for (int j = 0; j < n; j += kTileRows)
      a.tile[tile++] = {i < a.pool.adapters ? i : -1, at + j, min(n - j, kTileRows)};
    at += n;
  }
  for (int i = all + threadIdx.x; i < a.tiles; i += kGroupThreads)
    a.tile[i] = {-1, 0, 0};
  __syncthreads();
  for (int row = threadIdx.x; row < (a.rows + 63) / 64 * 64; row += kGroupThreads)
    add(row, true);
}

// Few rows are not sorted: each is a tile.
__device__ inline Tile tile_at(const AdapterArgs &a, int index) {
  if (!a.direct)
    return a.tile[index];
  const int adapter = checked_adapter(a, index);
  return {adapter < a.pool.adapters ? adapter : -1, index, 1};
}
__device__ inline int row_at(const AdapterArgs &a, int place) {
  return a.direct ? place : a.order[place];
}

// --------------------------------------------------------------- inner values
__device__ inline bf16x8 load8(const uint16_t *from) {
  return *reinterpret_cast<const bf16x8 *>(from);
}

// D (16 ranks) x X^T (16 rows) of every fourth 32-step of a part, for kCols 16s of rows and
// kRanks 16s of ranks. Lane l: row l % 16, ranks 4 (l / 16) + i. kAhead steps' operands are
// requested at once.
template <int kRanks, int kCols, bool kLow>
__device__ inline void down_tile(const AdapterArgs &a, const Tile &tile, int part,
                                 f32x4 (*sums)[kRanks * 4][64]) {
  constexpr int kLoads = kRanks + (kLow ? 2 : 1) * kCols;
  constexpr int kAhead = kLoads <= 3 ? 8 : kLoads <= 6 ? 4 : kLoads <= 12 ? 2 : 1;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rank = rank_of(a.pool, tile.adapter), width = a.pool.in_width;
  const uint16_t *down = a.pool.down + tile.adapter * a.pool.down_stride;
  // (Ranks that the adapter does not have take its first row; their sums are dropped.)
  const uint16_t *weight[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
    weight[r] = down + static_cast<size_t>(16 * r + col < rank ? 16 * r + col : 0) * width + 8 * g;
  size_t from[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    from[c] = row_at(a, tile.first + min(16 * c + col, tile.count - 1)) * a.x_stride + 8 * g;
  f32x4 sum[kRanks][kCols];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      sum[r][c] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};

  struct Step {
    bf16x8 weight[kRanks], hi[kCols], lo[kCols];
  };
  const auto load = [&](int k, Step &x) {
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
      x.weight[r] = load8(weight[r] + k);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      x.hi[c] = load8(a.hi + from[c] + k);
      if constexpr (kLow)
        x.lo[c] = load8(a.lo + from[c] + k);
    }
  };
  const auto add = [&](const Step &x) {
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        sum[r][c] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.weight[r], x.hi[c], sum[r][c], 0, 0, 0);
        if constexpr (kLow)
          sum[r][c] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.weight[r], x.lo[c], sum[r][c], 0, 0, 0);
      }
  };
  const int whole = width / 32, each = (whole + a.parts - 1) / a.parts;
  const int last = min(whole, (part + 1) * each);
  int step = part * each + wave;
  for (; step + 4 * (kAhead - 1) < last; step += 4 * kAhead) {
    Step x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      load(32 * (step + 4 * u), x[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      add(x[u]);
  }
  for (; step < last; step += 4) {
    Step x;
    load(32 * step, x);
    add(x);
  }
  if (width % 32 != 0 && part == a.parts - 1 && wave == 0) {
    // The last step ends inside: zeros in both operands, as zero times infinity is none.
    Step x{};
    if (32 * whole + 8 * g < width)
      load(32 * whole, x);
    add(x);
  }
  // The four waves' sums, always in the same order.
#pragma unroll
  for (int half = 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          sums[wave - half][r * kCols + c][lane] = sum[r][c];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          sum[r][c] += sums[wave][r * kCols + c][lane];
    }
    __syncthreads();
  }
  if (wave != 0)
    return;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    if (16 * c + col >= tile.count)
      continue;
    const int row = row_at(a, tile.first + 16 * c + col);
    float *inner = a.inner + (static_cast<size_t>(part) * a.rows + row) * a.pool.rank;
#pragma unroll
    for (int r = 0; r < kRanks; ++r) {
      const int first = 16 * r + 4 * g;
      if (first >= a.pool.rank)
        continue;
      f32x4 v = sum[r][c];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = first + i < rank ? v[i] : 0.0F;
      *reinterpret_cast<f32x4 *>(inner + first) = v;
    }
  }
}

template <int kRanks, bool kLow>
__global__ __launch_bounds__(256) void down_kernel(const AdapterArgs a) {
  __shared__ f32x4 sums[2][kRanks * 4][64];
  const Tile tile = tile_at(a, blockIdx.x / a.parts);
  if (tile.count == 0 || tile.adapter < 0)
    return;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  if (tile.count <= 16)
    down_tile<kRanks, 1, kLow>(a, tile, part, sums);
  else
    down_tile<kRanks, 4, kLow>(a, tile, part, sums);
}

// ------------------------------------------------------------------- outputs
// The three BF16 planes of values: 8 of their 24 bits each, by truncation, so exact.
__device__ inline void planes_of(const float (&v)[8], bf16x8 (&planes)[3]) {
  uint32_t word[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t part[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = v[2 * j + e];
      const uint32_t bits = __builtin_bit_cast(uint32_t, x);
      const float high = __builtin_bit_cast(float, bits & 0xffff0000U);
      const uint32_t rest = __builtin_bit_cast(uint32_t, x - high);
      const float middle = __builtin_bit_cast(float, rest & 0xffff0000U);
      // An infinity or NaN is in the first plane alone (a NaN with its quiet bit).
      const bool finite = (bits & 0x7f800000U) != 0x7f800000U;
      part[0][e] = finite || (bits & 0x7fffffU) == 0 ? bits : bits | 0x400000U;
      part[1][e] = finite ? rest : 0;
      part[2][e] = finite ? __builtin_bit_cast(uint32_t, x - high - middle) : 0;
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
      word[p][j] = __builtin_amdgcn_perm(part[p][1], part[p][0], 0x07060302U);
  }
#pragma unroll
  for (int p = 0; p < 3; ++p)
    __builtin_memcpy(&planes[p], word[p], 16);
}

// Rows without an adapter: their residual, or zero.
template <bool kVector, bool kResidual>
__device__ inline void copy_rows(const AdapterArgs &a, const Tile &tile, int begin, int last) {
  constexpr int kEach = kVector ? 4 : 1, kAhead = 8;
  typedef float vector __attribute__((ext_vector_type(kEach)));
  const int across = (last - begin) / kEach, all = tile.count * across;
  for (int first = threadIdx.x; first < all; first += 256 * kAhead) {
    size_t at[kAhead];
    vector v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(first + 256 * u, all - 1);
      at[u] = row_at(a, tile.first + i / across) * a.out_stride + begin + i % across * kEach;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      v[u] = 0.0F;
      if constexpr (kResidual)
        v[u] = *reinterpret_cast<const vector *>(a.residual + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (first + 256 * u < all)
        *reinterpret_cast<vector *>(a.out + at[u]) = v[u];
  }
}

// The inner values of 16 rows, summed over the parts, scaled and cut into planes: lane l
// holds row l % 16, ranks 8 (l / 16) .. of each 32-step. Zero behind the adapter's rank.
template <int kSteps> struct Inner {
  bf16x8 plane[kSteps][3];
  __device__ Inner(const AdapterArgs &a, int adapter, int rank, int row) {
    const int g = (threadIdx.x & 63) >> 4;
    const float scale = a.pool.scales == nullptr ? 1.0F : a.pool.scales[adapter];
    const size_t part_size = static_cast<size_t>(a.rows) * a.pool.rank;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = 32 * s + 8 * g;
      const float *source =
          a.inner + static_cast<size_t>(row) * a.pool.rank + (k < rank ? k : 0);
      f32x4 low{0.0F, 0.0F, 0.0F, 0.0F}, high = low;
#pragma unroll 4
      for (int part = 0; part < a.parts; ++part) {
        low += *reinterpret_cast<const f32x4 *>(source + part * part_size);
        high += *reinterpret_cast<const f32x4 *>(source + part * part_size + 4);
      }
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = k + e < rank ? (e < 4 ? low[e % 4] : high[e % 4]) * scale : 0.0F;
      planes_of(v, plane[s]);
    }
  }
};
// Clears the weights behind the adapter's rank, which may hold anything.
template <int kSteps> struct RankMask {
  uint32_t word[kSteps][4];
  __device__ explicit RankMask(int rank) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 32 * s + 8 * g + 2 * j;
        word[s][j] = (k < rank ? 0xffffU : 0U) | (k + 1 < rank ? 0xffff0000U : 0U);
      }
  }
  __device__ bf16x8 apply(const bf16x8 &weight, int s) const {
    uint32_t words[4];
    __builtin_memcpy(words, &weight, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      words[j] &= word[s][j];
    bf16x8 masked;
    __builtin_memcpy(&masked, words, 16);
    return masked;
  }
};

// U (16 columns) x inner^T (16 rows): lane l has row l % 16, columns 4 (l / 16) + i. The
// smallest plane first.
template <int kSteps>
__device__ inline f32x4 up_product(const bf16x8 (&weight)[kSteps], const Inner<kSteps> &inner) {
  f32x4 sum{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
  for (int p = 2; p >= 0; --p)
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(weight[s], inner.plane[s][p], sum, 0, 0, 0);
  return sum;
}

// 16 rows a wave, from registers to registers, of every `stride`th 16 columns; kAhead
// columns' operands are requested at once, by every lane from inside the tensors.
template <int kSteps, bool kVector, bool kResidual>
__device__ inline void up_rows(const AdapterArgs &a, const Tile &tile, int set, int n0, int stride,
                               int last) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int width = a.pool.out_width, rank = rank_of(a.pool, tile.adapter);
  const uint16_t *up = a.pool.up + tile.adapter * a.pool.up_stride;
  const bool mine = 16 * set + col < tile.count;
  const int row = row_at(a, tile.first + min(16 * set + col, tile.count - 1));
  const size_t at = row * a.out_stride;
  const Inner<kSteps> inner(a, tile.adapter, rank, row);
  const RankMask<kSteps> mask(rank);
  int from[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    from[s] = 32 * s + 8 * g < rank ? 32 * s + 8 * g : 0;

  struct Columns {
    bf16x8 weight[kSteps];
    f32x4 base;
  };
  const auto load = [&](int n, Columns &x) {
    const size_t column = min(n + col, width - 1);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      x.weight[s] = load8(up + column * a.pool.rank + from[s]);
    if constexpr (!kResidual) {
      x.base = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
    } else if constexpr (kVector) {
      x.base = *reinterpret_cast<const f32x4 *>(a.residual + at + min(n + 4 * g, width - 4));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.base[i] = a.residual[at + min(n + 4 * g + i, width - 1)];
    }
  };
  const auto finish = [&](int n, Columns &x) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      x.weight[s] = mask.apply(x.weight[s], s);
    const f32x4 v = up_product<kSteps>(x.weight, inner) + x.base;
    if (!mine)
      return;
    float *out = a.out + at + n + 4 * g;
    if constexpr (kVector) {
      if (n + 4 * g < last)
        *reinterpret_cast<f32x4 *>(out) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + 4 * g + i < last)
          out[i] = v[i];
    }
  };
  for (; n0 + (kAhead - 1) * stride < last; n0 += kAhead * stride) {
    Columns x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      load(n0 + u * stride, x[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      finish(n0 + u * stride, x[u]);
  }
  for (; n0 < last; n0 += stride) {
    Columns x;
    load(n0, x);
    finish(n0, x);
  }
}

// Tiles of more than 16 rows: a block takes 128 columns at a time, a wave 16 rows of them.
// The columns' weights pass through LDS for the four waves, the next ones on their way
// meanwhile; so do a wave's products, which it adds to the residual in whole runs of 512
// bytes of a row.
constexpr int kWide = 128;
template <int kSteps> struct WideShared {
  // (16 bytes more a row: neighbouring rows start on other banks.)
  __attribute__((aligned(16))) uint16_t weight[kWide][32 * kSteps + 8];
  __attribute__((aligned(16))) float product[kTileRows][kWide + 4];
};
template <int kSteps, bool kResidual>
__device__ inline void up_wide(const AdapterArgs &a, const Tile &tile, int begin, int last,
                               WideShared<kSteps> &shared) {
  constexpr int kPieces = kWide * 4 * kSteps / 256;  // 16 bytes of weights a thread
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int width = a.pool.out_width, rank = rank_of(a.pool, tile.adapter);
  const uint16_t *up = a.pool.up + tile.adapter * a.pool.up_stride;
  const int row = row_at(a, tile.first + min(16 * wave + col, tile.count - 1));
  const Inner<kSteps> inner(a, tile.adapter, rank, row);
  const RankMask<kSteps> mask(rank);
  const int rows = min(16, tile.count - 16 * wave);  // (0 and below: none)
  // Two rows of 32 lanes at a time.
  size_t at[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    at[i] = __shfl(row, 2 * i + (lane >> 5), 64) * a.out_stride;
  const int quad = lane % 32 * 4;

  bf16x8 piece[kPieces];
  const auto request = [&](int n0) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int i = threadIdx.x + 256 * j, k = i % (4 * kSteps) * 8;
      piece[j] = load8(up + static_cast<size_t>(min(n0 + i / (4 * kSteps), width - 1)) *
                                a.pool.rank + (k < a.pool.rank ? k : 0));
    }
  };
  request(begin);
  for (int n0 = begin; n0 < last; n0 += kWide) {
    __syncthreads();  // the last weights have been read
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int i = threadIdx.x + 256 * j;
      *reinterpret_cast<bf16x8 *>(&shared.weight[i / (4 * kSteps)][i % (4 * kSteps) * 8]) =
          piece[j];
    }
    __syncthreads();
    const int n = n0 + quad;
    f32x4 base[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      base[i] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
      if constexpr (kResidual)
        base[i] = *reinterpret_cast<const f32x4 *>(a.residual + at[i] + min(n, width - 4));
    }
    request(n0 + kWide);
    if (rows > 0) {
#pragma unroll
      for (int j = 0; j < kWide / 16; ++j) {
        bf16x8 weight[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          weight[s] = mask.apply(
              *reinterpret_cast<const bf16x8 *>(&shared.weight[16 * j + col][32 * s + 8 * g]), s);
        *reinterpret_cast<f32x4 *>(&shared.product[16 * wave + col][16 * j + 4 * g]) =
            up_product<kSteps>(weight, inner);
      }
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = 2 * i + (lane >> 5);
      const f32x4 v = *reinterpret_cast<const f32x4 *>(&shared.product[16 * wave + t][quad]);
      if (t < rows && n < last)
        *reinterpret_cast<f32x4 *>(a.out + at[i] + n) = base[i] + v;
    }
    wave_sync();
  }
}

template <int kSteps, bool kVector, bool kResidual>
__global__ __launch_bounds__(256) void up_kernel(const AdapterArgs a) {
  __shared__ std::conditional_t<kVector, WideShared<kSteps>, char> shared;
  const int chunks = (a.pool.out_width + a.chunk - 1) / a.chunk;
  const Tile tile = tile_at(a, blockIdx.x / chunks);
  if (tile.count == 0)
    return;
  const int begin = static_cast<int>(blockIdx.x % chunks) * a.chunk;
  const int last = min(a.pool.out_width, begin + a.chunk);
  if (tile.adapter < 0) {
    if (a.residual != a.out)
      copy_rows<kVector, kResidual>(a, tile, begin, last);
    return;
  }
  if constexpr (kVector) {
    if (tile.count > 16) {
      up_wide<kSteps, kResidual>(a, tile, begin, last, shared);
      return;
    }
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sets = tile.count <= 16 ? 1 : tile.count <= 32 ? 2 : 4;
  if (16 * (wave % sets) < tile.count)
    up_rows<kSteps, kVector, kResidual>(a, tile, wave % sets, begin + 16 * (wave / sets),
                                        64 / sets, last);
}

// ---------------------------------------------------------------------- host
// Tiles at most: each bin's last tile may be short.
size_t most_tiles(const AdapterPool &pool, size_t rows) {
  if (rows <= kDirectRows)
    return rows;
  return std::min(rows, rows / kTileRows + std::min<size_t>(rows, pool.adapters + size_t{1}));
}
// Parts of the width, so that a few tiles fill the card; eight 32-steps a wave at least.
size_t parts_of(const AdapterPool &pool, size_t rows) {
  const size_t steps = (static_cast<size_t>(pool.in_width) + 31) / 32;
  return std::max<size_t>(1, std::min<size_t>({16, 768 / most_tiles(pool, rows), steps / 32}));
}
size_t aligned(size_t bytes) { return (bytes + 15) / 16 * 16; }

template <int kRanks> void (*down_of(bool low))(AdapterArgs) {
  return low ? down_kernel<kRanks, true> : down_kernel<kRanks, false>;
}
template <int kSteps> void (*up_of(bool vector, bool residual))(AdapterArgs) {
  if (vector)
    return residual ? up_kernel<kSteps, true, true> : up_kernel<kSteps, true, false>;
  return residual ? up_kernel<kSteps, false, true> : up_kernel<kSteps, false, false>;
}

Status invalid(const char *why) { return {ErrorCode::kInvalidArgument, why}; }

}  // namespace

size_t adapter_workspace_bytes(const AdapterPool &pool, size_t rows) {
  return 2 * aligned(rows * sizeof(int32_t)) + aligned(most_tiles(pool, rows) * sizeof(Tile)) +
         parts_of(pool, rows) * rows * pool.rank * sizeof(float);
}

Status adapter_linear(const AdapterPool &pool, const int32_t *adapter, const uint16_t *x_hi,
                      const uint16_t *x_lo, size_t x_stride, size_t rows, const float *residual,
                      float *out, size_t out_stride, void *workspace, size_t workspace_bytes,
                      hipStream_t stream) {
  if (adapter == nullptr || x_hi == nullptr || out == nullptr)
    return invalid("adapter_linear: null tensor");
  if (reinterpret_cast<uintptr_t>(adapter) % 4 != 0 ||
      (reinterpret_cast<uintptr_t>(x_hi) | reinterpret_cast<uintptr_t>(x_lo)) % 16 != 0 ||
      x_stride % 8 != 0 || x_stride < static_cast<size_t>(pool.in_width) ||
      x_stride > (size_t{1} << 40))
    return invalid("adapter_linear: rows of x have to start on 16 bytes and hold in_width");
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) % 4 != 0 ||
      out_stride < static_cast<size_t>(pool.out_width) || out_stride > (size_t{1} << 40))
    return invalid("adapter_linear: out_stride below out_width, or misaligned outputs");
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
      workspace_bytes < adapter_workspace_bytes(pool, rows))
    return invalid("adapter_linear: workspace too small or not aligned");
  const size_t tiles = most_tiles(pool, rows), parts = parts_of(pool, rows);
  // About four blocks a CU, in whole rounds of a block's four waves.
  const size_t width = static_cast<size_t>(pool.out_width);
  const size_t chunk =
      std::min<size_t>(2048, std::max<size_t>(1, width * tiles / 1024 / 64) * 64);
  const size_t chunks = (width + chunk - 1) / chunk;
  constexpr size_t kMostBlocks = ((size_t{1} << 32) - 1) / 256;
  if (tiles * parts > kMostBlocks || tiles * chunks > kMostBlocks)
    return invalid("adapter_linear: grid too large");
  char *const base = static_cast<char *>(workspace);
  const size_t list = aligned(rows * sizeof(int32_t));
  char *const after = base + 2 * list;
  const bool vector =
      (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) % 16 == 0 &&
      out_stride % 4 == 0 && width % 4 == 0;
  const AdapterArgs args{pool, adapter, x_hi, x_lo, x_stride, static_cast<int>(rows), residual,
                         out, out_stride, static_cast<int>(tiles), static_cast<int>(parts),
                         static_cast<int>(chunk), rows <= kDirectRows ? 1 : 0,
                         reinterpret_cast<int32_t *>(base),
                         reinterpret_cast<int32_t *>(base + list), reinterpret_cast<Tile *>(after),
                         reinterpret_cast<float *>(after + aligned(tiles * sizeof(Tile)))};
  if (!args.direct)
    hipLaunchKernelGGL(group_kernel, dim3(1), dim3(kGroupThreads),
                       static_cast<unsigned>((pool.adapters + 1) * sizeof(int32_t)), stream,
                       args);
  const auto down = pool.rank <= 16   ? down_of<1>(x_lo != nullptr)
                    : pool.rank <= 32 ? down_of<2>(x_lo != nullptr)
                    : pool.rank <= 64 ? down_of<4>(x_lo != nullptr)
                                      : down_of<8>(x_lo != nullptr);
  hipLaunchKernelGGL(down, dim3(static_cast<unsigned>(tiles * parts)), dim3(256), 0, stream, args);
  const auto up = pool.rank <= 32   ? up_of<1>(vector, residual != nullptr)
                  : pool.rank <= 64 ? up_of<2>(vector, residual != nullptr)
                                    : up_of<4>(vector, residual != nullptr);
  hipLaunchKernelGGL(up, dim3(static_cast<unsigned>(tiles * chunks)), dim3(256), 0, stream, args);
  return launch_status("adapter_linear kernels");
}

}  // namespace evo::hip
