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
#include "ops.hpp"

#include <algorithm>

namespace evo::hip {

namespace {

constexpr int kTileRows = 64, kGroupThreads = 1024;

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
  int vector;   // output rows and columns in whole 16 bytes
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

// --------------------------------------------------------------- inner values
__device__ inline bf16x8 load_or_zero(const uint16_t *from, bool there) {
  bf16x8 v{};
  if (there)
    v = *reinterpret_cast<const bf16x8 *>(from);
  return v;
}

// D (16 ranks) x X^T (16 rows) of every fourth 32-step of a part, for kCols 16s of rows and
// kRanks 16s of ranks. Lane l: row l % 16, ranks 4 (l / 16) + i.
template <int kRanks, int kCols>
__device__ inline void down_tile(const AdapterArgs &a, const Tile &tile, int part,
                                 f32x4 (*sums)[kRanks * 4][64]) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rank = rank_of(a.pool, tile.adapter), width = a.pool.in_width;
  const uint16_t *down = a.pool.down + tile.adapter * a.pool.down_stride;
  const uint16_t *weight[kRanks];
  bool real[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r) {
    real[r] = 16 * r + col < rank;
    weight[r] = down + static_cast<size_t>(real[r] ? 16 * r + col : 0) * width + 8 * g;
  }
  size_t from[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int row = a.order[tile.first + min(16 * c + col, tile.count - 1)];
    from[c] = row * a.x_stride + 8 * g;
  }
  f32x4 sum[kRanks][kCols];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      sum[r][c] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
  const int steps = (width + 31) / 32, each = (steps + a.parts - 1) / a.parts;
  const int last = min(steps, (part + 1) * each);
  const bool low = a.lo != nullptr;
#pragma unroll 4
  for (int step = part * each + wave; step < last; step += 4) {
    const int k = 32 * step;
    const bool inside = k + 8 * g < width;
    bf16x8 w[kRanks], hi[kCols], lo[kCols];
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
      w[r] = load_or_zero(weight[r] + k, inside && real[r]);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      hi[c] = load_or_zero(a.hi + from[c] + k, inside);
      lo[c] = load_or_zero(a.lo + from[c] + k, inside && low);
    }
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        sum[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r], hi[c], sum[r][c], 0, 0, 0);
        if (low)
          sum[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r], lo[c], sum[r][c], 0, 0, 0);
      }
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
    const int row = a.order[tile.first + 16 * c + col];
    float *inner = a.inner + (static_cast<size_t>(part) * a.rows + row) * a.pool.rank;
#pragma unroll
    for (int r = 0; r < kRanks; ++r) {
      const int first = 16 * r + 4 * g;
      if (first >= a.pool.rank)
        continue;
      // (Behind the adapter's rank zeros met the row's values, infinities among them.)
      f32x4 v = sum[r][c];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = first + i < rank ? v[i] : 0.0F;
      *reinterpret_cast<f32x4 *>(inner + first) = v;
    }
  }
}

template <int kRanks>
__global__ __launch_bounds__(256) void down_kernel(const AdapterArgs a) {
  __shared__ f32x4 sums[2][kRanks * 4][64];
  const Tile tile = a.tile[blockIdx.x / a.parts];
  if (tile.count == 0 || tile.adapter < 0)
    return;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  if (tile.count <= 16)
    down_tile<kRanks, 1>(a, tile, part, sums);
  else
    down_tile<kRanks, 4>(a, tile, part, sums);
}

// ------------------------------------------------------------------- outputs
// Columns n .. n + 3 of a row.
__device__ inline f32x4 load_columns(const AdapterArgs &a, const float *row, int n) {
  f32x4 v{0.0F, 0.0F, 0.0F, 0.0F};
  if (row == nullptr)
    return v;
  if (a.vector) {
    if (n < a.pool.out_width)
      v = *reinterpret_cast<const f32x4 *>(row + n);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < a.pool.out_width)
      v[i] = row[n + i];
  return v;
}
__device__ inline void store_columns(const AdapterArgs &a, float *row, int n, const f32x4 &v) {
  if (a.vector) {
    if (n < a.pool.out_width)
      *reinterpret_cast<f32x4 *>(row + n) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < a.pool.out_width)
      row[n + i] = v[i];
}

// The three BF16 planes of a value: 8 of its 24 bits each, by truncation, so exact.
__device__ inline void planes_of(float v, uint16_t (&plane)[3]) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v);
  if ((bits & 0x7f800000U) == 0x7f800000U) {
    plane[0] = static_cast<uint16_t>(bits >> 16 | ((bits & 0x7fffffU) != 0 ? 0x40U : 0));
    plane[1] = plane[2] = 0;
    return;
  }
  const float high = __builtin_bit_cast(float, bits & 0xffff0000U);
  const uint32_t rest = __builtin_bit_cast(uint32_t, v - high);
  const float middle = __builtin_bit_cast(float, rest & 0xffff0000U);
  const float low = v - high - middle;
  plane[0] = static_cast<uint16_t>(bits >> 16);
  plane[1] = static_cast<uint16_t>(rest >> 16);
  plane[2] = static_cast<uint16_t>(__builtin_bit_cast(uint32_t, low) >> 16);
}

// U (16 columns) x inner^T (16 rows). Lane l: row l % 16, columns 4 (l / 16) + i.
template <int kSteps, int kCols, typename Planes>
__device__ inline void up_tile(const AdapterArgs &a, const Tile &tile, int chunk,
                               const Planes &planes) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rank = rank_of(a.pool, tile.adapter), width = a.pool.out_width;
  const uint16_t *up = a.pool.up + tile.adapter * a.pool.up_stride;
  size_t at[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    at[c] = a.order[tile.first + min(16 * c + col, tile.count - 1)] * a.out_stride;
  const int last = min(width, (chunk + 1) * a.chunk);
  for (int n0 = chunk * a.chunk + 16 * wave; n0 < last; n0 += 64) {
    bf16x8 w[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = 32 * s + 8 * g;
      w[s] = load_or_zero(up + static_cast<size_t>(n0 + col) * a.pool.rank + k,
                          n0 + col < width && k < rank);
      if (rank % 8 != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[s][e] = k + e < rank ? w[s][e] : static_cast<__bf16>(0.0F);
      }
    }
    const int n = n0 + 4 * g;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const bool mine = 16 * c + col < tile.count;
      const f32x4 base =
          load_columns(a, mine && a.residual != nullptr ? a.residual + at[c] : nullptr, n);
      f32x4 sum{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const bf16x8 h =
              *reinterpret_cast<const bf16x8 *>(&planes[p][16 * c + col][32 * s + 8 * g]);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[s], h, sum, 0, 0, 0);
        }
      if (mine)
        store_columns(a, a.out + at[c], n, base + sum);
    }
  }
}

template <int kSteps> __global__ __launch_bounds__(256) void up_kernel(const AdapterArgs a) {
  // (Rows of 16 bytes more: neighbouring rows start on other banks.)
  __shared__ __attribute__((aligned(16))) uint16_t planes[3][kTileRows][32 * kSteps + 8];
  const int chunks = (a.pool.out_width + a.chunk - 1) / a.chunk;
  const Tile tile = a.tile[blockIdx.x / chunks];
  const int chunk = static_cast<int>(blockIdx.x % chunks);
  if (tile.count == 0)
    return;
  if (tile.adapter < 0) {
    if (a.residual == a.out)
      return;
    const int quads = a.chunk / 4;
    for (int i = threadIdx.x; i < tile.count * quads; i += 256) {
      const size_t at = a.order[tile.first + i / quads] * a.out_stride;
      const int n = chunk * a.chunk + i % quads * 4;
      store_columns(a, a.out + at, n,
                    load_columns(a, a.residual != nullptr ? a.residual + at : nullptr, n));
    }
    return;
  }
  const float scale = a.pool.scales == nullptr ? 1.0F : a.pool.scales[tile.adapter];
  constexpr int kQuads = 8 * kSteps;
  for (int i = threadIdx.x; i < tile.count * kQuads; i += 256) {
    const int t = i / kQuads, k = i % kQuads * 4;
    f32x4 v{0.0F, 0.0F, 0.0F, 0.0F};
    if (k < a.pool.rank) {
      const int row = a.order[tile.first + t];
      const float *inner = a.inner + static_cast<size_t>(row) * a.pool.rank + k;
      for (int part = 0; part < a.parts; ++part)
        v += *reinterpret_cast<const f32x4 *>(inner + static_cast<size_t>(part) * a.rows *
                                                          a.pool.rank);
    }
    uint16_t cut[4][3];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      planes_of(v[e] * scale, cut[e]);
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<ushort4 *>(&planes[p][t][k]) =
          make_ushort4(cut[0][p], cut[1][p], cut[2][p], cut[3][p]);
  }
  __syncthreads();
  if (tile.count <= 16)
    up_tile<kSteps, 1>(a, tile, chunk, planes);
  else
    up_tile<kSteps, 4>(a, tile, chunk, planes);
}

// ---------------------------------------------------------------------- host
// Tiles at most: each bin's last tile may be short.
size_t most_tiles(const AdapterPool &pool, size_t rows) {
  return std::min(rows, rows / kTileRows + std::min<size_t>(rows, pool.adapters + size_t{1}));
}
// Parts of the width, so that a few tiles fill the card; two 32-steps a wave at least.
size_t parts_of(const AdapterPool &pool, size_t rows) {
  const size_t steps = (static_cast<size_t>(pool.in_width) + 31) / 32;
  return std::max<size_t>(1, std::min<size_t>({16, 768 / most_tiles(pool, rows), steps / 8}));
}
size_t aligned(size_t bytes) { return (bytes + 15) / 16 * 16; }

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
                         static_cast<int>(chunk), vector ? 1 : 0,
                         reinterpret_cast<int32_t *>(base),
                         reinterpret_cast<int32_t *>(base + list), reinterpret_cast<Tile *>(after),
                         reinterpret_cast<float *>(after + aligned(tiles * sizeof(Tile)))};
  hipLaunchKernelGGL(group_kernel, dim3(1), dim3(kGroupThreads),
                     static_cast<unsigned>((pool.adapters + 1) * sizeof(int32_t)), stream, args);
  const auto down = pool.rank <= 16   ? down_kernel<1>
                    : pool.rank <= 32 ? down_kernel<2>
                    : pool.rank <= 64 ? down_kernel<4>
                                      : down_kernel<8>;
  hipLaunchKernelGGL(down, dim3(static_cast<unsigned>(tiles * parts)), dim3(256), 0, stream, args);
  const auto up = pool.rank <= 32 ? up_kernel<1> : pool.rank <= 64 ? up_kernel<2> : up_kernel<4>;
  hipLaunchKernelGGL(up, dim3(static_cast<unsigned>(tiles * chunks)), dim3(256), 0, stream, args);
  return launch_status("adapter_linear kernels");
}

}  // namespace evo::hip
