// SPDX-License-Identifier: Apache-2.0
// Low-rank adapters of many requests beside a shared product:
//   out[t] = residual[t] + s_a U_a (D_a x[t]),  a the adapter of row t (or none).
//
// Rows are sorted by adapter on the device, so that an adapter is read once for up to 64
// of its rows wherever they lie: by group_kernel, or where they are few enough by each block
// of down_kernel for itself. down_kernel forms the inner values D_a x of such a tile for a part
// of the width, up_kernel adds the parts up, scales them and forms a chunk of the output
// columns. Two launches, as the second product needs all of the width; both_kernel takes calls
// of little work in one.
// x comes as the planes hi (+ lo) of a split-BF16 activation, whose products with BF16
// weights are exact in F32. The inner values are F32, and stay so in the second product:
// each is cut into three BF16 planes, 8 bits each, which hold all of its 24 (one plane
// would round them to 2^-9, and the update with them; the two more cost matrix
// instructions, which are not what bounds it). An infinity in U meets the planes that are zero
// too, and gives NaN; both_kernel, which has no planes, gives the infinity.
// A row's values come from its own column of each product: an infinity or NaN of one row
// or adapter reaches no other row.
//
// What bounds it. Many rows: bytes, nearly all of them the residual and the outputs. 4096
// prompt rows on 8 adapters of rank 64, width 4096 -> 12288 (481 MB): first product 29 us, 5
// of them the sort (67 MB of x), second 78 (403 MB and weights, 5.2 TB/s, a copy's rate). Few
// rows: the chain of launch, sort and loads that wait for each other. 512 rows of 6 adapters
// of rank 64, width 4096 -> 11264: 7.8 + 16.5 us (62 MB, 12.2 us of a copy); in one launch one
// row of rank 16 6.2 us, 96 rows of 40 adapters 13.4 (30 MB, 5.9).
#include "common.hpp"
#include "lanes.hpp"
#include "ops.hpp"

#include <algorithm>
#include <type_traits>

namespace evo::hip {

namespace {

constexpr int kTileRows = 64, kGroupThreads = 1024;
constexpr int kSingleRows = 4;   // up to these, each row is a tile of its own
constexpr int kFewRows = 512;    // up to these the tiles found say how work is divided
constexpr int kSelfRows = 4096;  // up to these blocks of down_kernel may sort for themselves
constexpr int kMostSorts = 640;  // blocks that do at most
constexpr int kManyRows = 2048;  // from these on work is divided by the tiles expected

struct Tile {
  int adapter, first, count;  // rows order[first ..]; adapter -1: rows without one
  int parts;                  // that its inner values come in
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
  int parts;    // of the width at most, in down_kernel
  int chunk;    // output columns of a block, in up_kernel
  int sorted;   // by group_kernel
  int halves;   // blocks of down_kernel that share a tile's rows, 32 at a time
  int wide;     // tiles of more than 16 rows go through LDS in up_kernel
  int narrow;   // up_kernel divides its columns by the tiles found, 256 at most
  int32_t *bin;    // [rows], the adapter of each as it was read; the pool's size: none
  int32_t *order;  // rows sorted by it; kTileRows for each tile, where down_kernel sorts
  int places;      // in order
  Tile *tile;      // [tiles], count 0 behind the last
  int32_t *found;  // how many tiles there are
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
// those without. A thread's first kKept rows are requested at once and kept. 4096 rows
// take 7.6 us, most of it the launch, one load and the additions to bins in LDS; more
// blocks would have to count together, which takes a launch more.
constexpr int kKept = 8;
__global__ __launch_bounds__(kGroupThreads) void group_kernel(const AdapterArgs a) {
  extern __shared__ int32_t bins[];
  __shared__ int32_t rows_before[kGroupThreads / 64], tiles_before[kGroupThreads / 64];
  const int threads = static_cast<int>(blockDim.x), waves = threads / 64;
  const int count = a.pool.adapters + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int kept[kKept];
#pragma unroll
  for (int j = 0; j < kKept; ++j) {
    const int row = threadIdx.x + j * threads;
    kept[j] = row < a.rows ? checked_adapter(a, row) : -1;
  }
  for (int i = threadIdx.x; i < count; i += threads)
    bins[i] = 0;
  __syncthreads();
  // The place of a wave's rows (bin -1: none) in their bins: one addition where all of
  // them share one, as in prompts.
  const auto add = [&](int bin) {
    const int first = __builtin_amdgcn_readfirstlane(bin);
    const uint64_t same = __ballot(bin == first);
    if (first >= 0 && same == __ballot(bin >= 0)) {
      int at = 0;
      if (lane == 0)
        at = atomicAdd(&bins[first], static_cast<int>(__popcll(same)));
      return __builtin_amdgcn_readfirstlane(at) + lane;
    }
    return bin < 0 ? 0 : atomicAdd(&bins[bin], 1);
  };
#pragma unroll
  for (int j = 0; j < kKept; ++j)
    if (j * threads < a.rows)
      add(kept[j]);
  // (Rows beyond those are read once too: both passes see one adapter.)
  for (int first = kKept * threads; first < a.rows; first += threads) {
    const int row = first + threadIdx.x;
    const int bin = row < a.rows ? checked_adapter(a, row) : -1;
    if (row < a.rows)
      a.bin[row] = bin;
    add(bin);
  }
  __syncthreads();

  // Each thread's bins, and what lies before them.
  const int each = (count + threads - 1) / threads, from = threadIdx.x * each;
  int rows = 0, tiles = 0;
  for (int i = from; i < min(from + each, count); ++i) {
    rows += bins[i];
    tiles += (bins[i] + kTileRows - 1) / kTileRows;
  }
  const int rows_through = wave_scan<Sum>(rows), tiles_through = wave_scan<Sum>(tiles);
  if (lane == 63) {
    rows_before[wave] = rows_through;
    tiles_before[wave] = tiles_through;
  }
  __syncthreads();
  int at = rows_through - rows, tile = tiles_through - tiles, all = 0;
  for (int w = 0; w < waves; ++w) {
    at += w < wave ? rows_before[w] : 0;
    tile += w < wave ? tiles_before[w] : 0;
    all += tiles_before[w];
  }
  for (int i = from; i < min(from + each, count); ++i) {
    const int n = bins[i];
    bins[i] = at;
    for (int j = 0; j < n; j += kTileRows)
      a.tile[tile++] = {i < a.pool.adapters ? i : -1, at + j, min(n - j, kTileRows), a.parts};
    at += n;
  }
  for (int i = all + threadIdx.x; i < a.tiles; i += threads)
    a.tile[i] = {-1, 0, 0, 0};
  if (threadIdx.x == 0)
    *a.found = all;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kKept; ++j)
    if (j * threads < a.rows) {
      const int place = add(kept[j]);
      if (kept[j] >= 0)
        a.order[place] = static_cast<int32_t>(threadIdx.x + j * threads);
    }
  for (int first = kKept * threads; first < a.rows; first += threads) {
    const int row = first + threadIdx.x;
    const int bin = row < a.rows ? max(0, min(a.bin[row], count - 1)) : -1;
    const int place = add(bin);
    if (row < a.rows && place < a.rows)
      a.order[place] = row;
  }
}

// A block's tile: its rows in list[0 .. count).
struct TileRows {
  Tile tile;
  int list[kTileRows];
};
// A tile of the list. What stands there is bounded before it is followed: a workspace that
// someone else writes meanwhile costs the call its values and no more.
__device__ inline Tile checked_tile(const AdapterArgs &a, const Tile &tile) {
  if (tile.adapter < -1 || tile.adapter >= a.pool.adapters || tile.count < 0 ||
      tile.count > kTileRows || tile.first < 0 || tile.first > a.places - tile.count ||
      tile.parts < 0 || tile.parts > a.parts)
    return {-1, 0, 0, 0};
  return tile;
}
__device__ inline void find_rows(const AdapterArgs &a, const Tile &tile, TileRows &s) {
  if (static_cast<int>(threadIdx.x) < tile.count)
    s.list[threadIdx.x] = max(0, min(a.order[tile.first + threadIdx.x], a.rows - 1));
}
__device__ inline void find_tile(const AdapterArgs &a, int index, TileRows &s) {
  const Tile tile = checked_tile(a, a.tile[index]);
  find_rows(a, tile, s);
  if (threadIdx.x == 0)
    s.tile = tile;
  __syncthreads();
}

// Rows are sorted by each block of down_kernel for itself where that takes it less than a
// launch, 5 to 8 us: it counts the adapters' rows, so the tiles of each, finds the adapter
// of its own tile, and in row order that adapter's rows. The number of tiles says into how
// many parts the blocks divide the width.
constexpr int kDownWaves = 8, kCus = 256;
constexpr int kUsualWidth = 32 * 4 * kDownWaves;  // of a part: four steps a wave
constexpr int kOwnRows = kSelfRows / (64 * kDownWaves);
struct Counts {
  int tiles[kDownWaves], words[kSelfRows / 64];
};
static_assert(kSelfRows / 64 <= 64, "a wave adds up the words' counts");
// What a block of down_kernel takes: a tile (its rows in TileRows), up to 32 of its rows
// from 16 set, up to 16 group_ranks of its ranks and a part of the width.
struct DownWork {
  int tiles, parts, group_ranks, index, set, group, part;
};
// How the blocks share `tiles` tiles: parts of the width, about four steps a wave, or two
// where that leaves half the card (301 rows of 9 adapters of width 1920 16.4 us for 17.5, but
// 300 rows of 40 21.3 for 19.9).
// And where parts leave half the card, 32 ranks a block rather than 64: each reads x, but half
// as many weights one after the other (512 rows of 6 adapters of rank 64 25.1 us for 26.3,
// 182 rows of 2 of rank 88 18.6 for 21.5; 460 rows of 16 of rank 40 and width 11264, which
// fill the card, 35.0 for 31.7).
__device__ inline DownWork down_work(const AdapterArgs &a, int tiles, int kernel_ranks) {
  int ranks = kernel_ranks, groups = 1, parts = a.parts;
  if (a.rows <= kFewRows) {
    const int all = (a.pool.rank + 15) / 16, units = max(1, tiles) * a.halves;
    const auto divide = [&](int of_block) {
      ranks = of_block;
      groups = (all + ranks - 1) / ranks;
      const int usual = min(a.parts, (a.pool.in_width + kUsualWidth - 1) / kUsualWidth);
      parts = max(usual, min(a.parts, kCus / (units * groups)));
      parts = max(1, min(parts, static_cast<int>(gridDim.x) / (units * groups)));
    };
    divide(min(kernel_ranks, 2));
    if (kernel_ranks > 2 && units * groups * parts > kCus)
      divide(kernel_ranks);
  }
  const int unit = static_cast<int>(blockIdx.x) / parts, half = unit / groups;
  return {tiles, parts, ranks, half / a.halves, half % a.halves * 2, unit % groups,
          static_cast<int>(blockIdx.x) % parts};
}
__device__ inline DownWork sort_tile(const AdapterArgs &a, int kernel_ranks, Counts &counts,
                                     int32_t *bins, TileRows &s) {
  constexpr int kThreads = 64 * kDownWaves;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int count = a.pool.adapters + 1;
  int own[kOwnRows];
#pragma unroll
  for (int j = 0; j < kOwnRows; ++j) {
    const int row = threadIdx.x + j * kThreads;
    own[j] = row < a.rows ? checked_adapter(a, row) : -1;
  }
  for (int i = threadIdx.x; i < count; i += kThreads)
    bins[i] = 0;
  if (threadIdx.x == 0)
    s.tile = {-1, 0, 0, 0};
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kOwnRows; ++j) {
    if (j * kThreads >= a.rows)
      break;
    // One addition where all of a wave's rows share an adapter, as in prompts.
    const int first = __builtin_amdgcn_readfirstlane(own[j]);
    const uint64_t same = __ballot(own[j] == first);
    if (first >= 0 && same == __ballot(own[j] >= 0)) {
      if (lane == 0)
        atomicAdd(&bins[first], static_cast<int>(__popcll(same)));
    } else if (own[j] >= 0) {
      atomicAdd(&bins[own[j]], 1);
    }
  }
  __syncthreads();
  const int each = (count + kThreads - 1) / kThreads, from = threadIdx.x * each;
  int mine = 0;
  for (int i = from; i < min(from + each, count); ++i)
    mine += (bins[i] + kTileRows - 1) / kTileRows;
  const int through = wave_scan<Sum>(mine);
  if (lane == 63)
    counts.tiles[wave] = through;
  __syncthreads();
  int at = through - mine, tiles = 0;  // tiles of the bins before this thread's, and all
#pragma unroll
  for (int w = 0; w < kDownWaves; ++w) {
    at += w < wave ? counts.tiles[w] : 0;
    tiles += counts.tiles[w];
  }
  const DownWork work = down_work(a, tiles, kernel_ranks);
  if (at <= work.index && work.index < at + mine) {
    int bin = from, first = (work.index - at) * kTileRows;
    for (; first >= bins[bin]; ++bin)
      first -= (bins[bin] + kTileRows - 1) / kTileRows * kTileRows;
    s.tile = {bin, first, min(bins[bin] - first, kTileRows), work.parts};
  }
  __syncthreads();
  const Tile tile = s.tile;
  if (tile.count == 0)
    return work;
  uint64_t same[kOwnRows];
#pragma unroll
  for (int j = 0; j < kOwnRows; ++j) {
    if (j * kThreads >= a.rows)
      break;
    same[j] = __ballot(own[j] == tile.adapter);
    if (lane == 0)
      counts.words[wave + j * kDownWaves] = __popcll(same[j]);
  }
  __syncthreads();
  const int here = 64 * lane < a.rows ? counts.words[lane] : 0;
  const int before = wave_scan<Sum>(here) - here;
#pragma unroll
  for (int j = 0; j < kOwnRows; ++j) {
    if (j * kThreads >= a.rows)
      break;
    const int place = __builtin_amdgcn_readlane(before, wave + j * kDownWaves) - tile.first +
                      __popcll(same[j] & ((uint64_t{1} << lane) - 1));
    if (own[j] == tile.adapter && place >= 0 && place < tile.count)
      s.list[place] = threadIdx.x + j * kThreads;
  }
  if (threadIdx.x == 0) {
    s.tile.first = work.index * kTileRows;
    if (tile.adapter == a.pool.adapters)
      s.tile.adapter = -1;
  }
  __syncthreads();
  return work;
}
// Up to 4 rows: each is a tile. (Rank 64, width 4096 -> 12288, us sorted and not: 4 rows of 4
// adapters 13.6 and 12.8, 8 rows of 2 13.3 and 16.9, 16 rows of 2 13.8 and 18.8, of 16 20.3
// and 19.3.)
__device__ inline DownWork single_tile(const AdapterArgs &a, int kernel_ranks, TileRows &s) {
  const DownWork work = down_work(a, a.rows, kernel_ranks);
  if (threadIdx.x == 0) {
    s.tile = {-1, 0, 0, 0};
    if (work.index < a.rows) {
      const int adapter = checked_adapter(a, work.index);
      s.tile = {adapter < a.pool.adapters ? adapter : -1, work.index * kTileRows, 1,
                work.parts};
      s.list[0] = work.index;
    }
  }
  __syncthreads();
  return work;
}

// --------------------------------------------------------------- inner values
__device__ inline bf16x8 load8(const uint16_t *from) {
  return *reinterpret_cast<const bf16x8 *>(from);
}

// D (16 ranks) x X^T (16 rows) of a part of the width, for the kCols 16s of rows from `set`
// on and kRanks 16s of ranks. Each wave takes every eighth 32-step, kAhead of them
// requested at once (with more, no faster); their sums meet in LDS.
// Loaded as the products take them, 16 neighbouring lanes would read 16 rows, which costs
// the load unit a cycle each (64 to 85 a load measured, 4096 rows 34 us). Four neighbouring
// lanes read 64 bytes of one row instead, and the wave turns them in LDS: lane l holds piece
// (l % 4) ^ (l / 8 % 4) of row l / 4 (so turned, neither side meets bank conflicts), and
// takes row l % 16, piece l / 16. Its sums are row l % 16, ranks 4 (l / 16) + i.
template <int kRanks, int kCols, bool kLow>
__device__ inline void down_tile(const AdapterArgs &a, const TileRows &rows, const DownWork &work,
                                 int set, f32x4 *shared) {
  const Tile &tile = rows.tile;
  constexpr int kLoads = kRanks + (kLow ? 2 : 1) * kCols;
  constexpr int kAhead = kLoads <= 6 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rank = rank_of(a.pool, tile.adapter), width = a.pool.in_width;
  const uint16_t *down = a.pool.down + tile.adapter * a.pool.down_stride;
  const int part = work.part, base = 16 * kRanks * work.group;
  if (base >= rank)
    return;
  // Row r of a load's 16 is at LDS place 4 r + (piece ^ r / 2 % 4).
  const int owner = lane >> 2, piece = (lane & 3) ^ (lane >> 3 & 3);
  const int taken = 4 * (lane & 15) + ((lane >> 4) ^ (lane >> 1 & 3));
  f32x4 *const turn = shared + wave * kLoads * 64;
  // (Ranks that the adapter does not have take its first row; their sums are dropped.)
  const uint16_t *weight[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
    weight[r] = down + static_cast<size_t>(base + 16 * r + owner < rank ? base + 16 * r + owner
                                                                        : 0) * width;
  size_t from[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    from[c] = rows.list[min(16 * (set + c) + owner, tile.count - 1)] * a.x_stride;
  f32x4 sum[kRanks][kCols];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      sum[r][c] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};

  const int steps = (width + 31) / 32, each = (steps + tile.parts - 1) / tile.parts;
  const int last = min(steps, (part + 1) * each);
  for (int step = part * each + wave; step < last; step += kDownWaves * kAhead) {
    bf16x8 x[kAhead][kLoads];  // weights, hi and lo planes
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = 32 * min(step + kDownWaves * u, steps - 1) + 8 * piece;
      const int k = at < width ? at : 0;
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
        x[u][r] = load8(weight[r] + k);
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        x[u][kRanks + c] = load8(a.hi + from[c] + k);
        if constexpr (kLow)
          x[u][kRanks + kCols + c] = load8(a.lo + from[c] + k);
      }
    }
    asm volatile("" ::: "memory");  // every load before the first product
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = step + kDownWaves * u;
      if (at >= last)
        break;
      // Behind the width: zeros in both operands, as zero times infinity is none.
      const bool there = 32 * at + 8 * piece < width;
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        turn[64 * j + lane] = there ? __builtin_bit_cast(f32x4, x[u][j]) : f32x4{};
      wave_sync();
      bf16x8 v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        v[j] = __builtin_bit_cast(bf16x8, turn[64 * j + taken]);
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          sum[r][c] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[r], v[kRanks + c], sum[r][c], 0, 0, 0);
          if constexpr (kLow)
            sum[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[r], v[kRanks + kCols + c],
                                                                sum[r][c], 0, 0, 0);
        }
      wave_sync();
    }
  }
  __syncthreads();
  f32x4 *const sums = shared;
  constexpr int kSums = kRanks * kCols * 64;  // of a wave
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      sums[wave * kSums + (r * kCols + c) * 64 + lane] = sum[r][c];
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < kSums; i += 64 * kDownWaves) {
    f32x4 v = sums[i];
#pragma unroll
    for (int w = 1; w < kDownWaves; ++w)
      v += sums[w * kSums + i];
    const int t = 16 * (set + i / 64 % kCols) + i % 16;
    const int first = base + 16 * (i / 64 / kCols) + 4 * (i % 64 / 16);
    if (t >= tile.count || first >= a.pool.rank)
      continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = first + e < rank ? v[e] : 0.0F;
    const size_t row = static_cast<size_t>(part) * a.rows + rows.list[t];
    *reinterpret_cast<f32x4 *>(a.inner + row * a.pool.rank + first) = v;
  }
}

// A block takes up to 32 rows of a tile at a time and a part of the width.
template <int kRanks, bool kLow>
__global__ __launch_bounds__(64 * kDownWaves) void down_kernel(const AdapterArgs a) {
  extern __shared__ f32x4 down_shared[];
  __shared__ TileRows rows;
  __shared__ Counts counts;
  DownWork work;
  if (a.sorted) {
    work = down_work(a, a.tiles, kRanks);
    find_tile(a, work.index, rows);
  } else {
    work = a.rows <= kSingleRows ? single_tile(a, kRanks, rows)
                                 : sort_tile(a, kRanks, counts,
                                             reinterpret_cast<int32_t *>(down_shared), rows);
    // For up_kernel: this tile, and that there are none behind the last.
    if (rows.tile.count > 0 && work.part == 0 && work.set == 0 && work.group == 0) {
      if (static_cast<int>(threadIdx.x) < rows.tile.count)
        a.order[rows.tile.first + threadIdx.x] = rows.list[threadIdx.x];
      if (threadIdx.x == 0)
        a.tile[work.index] = rows.tile;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0)
      *a.found = work.tiles;
    if (blockIdx.x == 0)
      for (int i = work.tiles + static_cast<int>(threadIdx.x); i < a.tiles; i += blockDim.x)
        a.tile[i] = {-1, 0, 0, 0};
  }
  if (rows.tile.adapter < 0)
    return;
  const auto take = [&](auto ranks, int set) {
    if (rows.tile.count - 16 * set <= 16)
      down_tile<decltype(ranks)::value, 1, kLow>(a, rows, work, set, down_shared);
    else
      down_tile<decltype(ranks)::value, 2, kLow>(a, rows, work, set, down_shared);
  };
#pragma unroll 1
  for (int set = work.set; 16 * set < rows.tile.count; set += 2 * a.halves) {
    if (kRanks == 4 && work.group_ranks == 2)
      take(std::integral_constant<int, 2>(), set);
    else
      take(std::integral_constant<int, kRanks>(), set);
    __syncthreads();
  }
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

// Output widths: of whole quads, not, and below one.
enum Width : int { kWhole, kRagged, kNarrow };
// Four columns of an output row, 16 bytes that may start anywhere a float may.
typedef f32x4 quad __attribute__((aligned(4)));
// Columns n .. n + 3 of a residual row of at least 4, whatever n: loaded from inside the row.
// `ends`: some lane's columns may pass its end, where a quad does not end.
__device__ inline f32x4 load_quad(const float *row, int n, int width, bool ends) {
  f32x4 v = *reinterpret_cast<const quad *>(row + min(n, width - 4));
  if (ends && n < width && n + 4 > width) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = row[min(n + i, width - 1)];
  }
  return v;
}
template <bool kStream>
__device__ inline void store_quad(float *row, int n, int width, bool ends, const f32x4 &v) {
  if (n + 4 <= width) {
    if constexpr (kStream)
      __builtin_nontemporal_store(v, reinterpret_cast<quad *>(row + n));
    else
      *reinterpret_cast<quad *>(row + n) = v;
  } else if (ends) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < width)
        row[n + i] = v[i];
  }
}

// Rows without an adapter: their residual, or zero.
template <bool kResidual>
__device__ inline void copy_rows(const AdapterArgs &a, const TileRows &rows, int begin,
                                 int last) {
  constexpr int kAhead = 8;
  const int across = (last - begin) / 4, all = rows.tile.count * across;
  for (int first = threadIdx.x; first < all; first += 256 * kAhead) {
    size_t at[kAhead];
    f32x4 v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(first + 256 * u, all - 1);
      at[u] = rows.list[i / across] * a.out_stride + begin + i % across * 4;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      v[u] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
      if constexpr (kResidual)
        v[u] = *reinterpret_cast<const quad *>(a.residual + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (first + 256 * u < all)
        *reinterpret_cast<quad *>(a.out + at[u]) = v[u];
  }
  // What no quad holds.
  const int rest = (last - begin) % 4;
  for (int i = threadIdx.x; i < rows.tile.count * rest; i += 256) {
    const size_t at = rows.list[i / rest] * a.out_stride + last - rest + i % rest;
    a.out[at] = kResidual ? a.residual[at] : 0.0F;
  }
}

// The inner values of 16 rows, summed over the parts, scaled and cut into planes: lane l
// holds row l % 16, ranks 8 (l / 16) .. of each 32-step. Zero behind the adapter's rank.
template <int kSteps> struct Inner {
  bf16x8 plane[kSteps][3];
  __device__ Inner(const AdapterArgs &a, const Tile &tile, int rank, int row) {
    const int g = (threadIdx.x & 63) >> 4;
    const float scale = a.pool.scales == nullptr ? 1.0F : a.pool.scales[tile.adapter];
    const size_t part_size = static_cast<size_t>(a.rows) * a.pool.rank;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = 32 * s + 8 * g;
      const float *source =
          a.inner + static_cast<size_t>(row) * a.pool.rank + (k < rank ? k : 0);
      f32x4 low{0.0F, 0.0F, 0.0F, 0.0F}, high = low;
#pragma unroll 4
      for (int part = 0; part < tile.parts; ++part) {
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
template <int kSteps, int kWidth, bool kResidual>
__device__ inline void up_rows(const AdapterArgs &a, const TileRows &rows, int set, int n0,
                               int stride, int last) {
  const Tile &tile = rows.tile;
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int width = a.pool.out_width, rank = rank_of(a.pool, tile.adapter);
  const uint16_t *up = a.pool.up + tile.adapter * a.pool.up_stride;
  const bool mine = 16 * set + col < tile.count;
  const int row = rows.list[min(16 * set + col, tile.count - 1)];
  const size_t at = row * a.out_stride;
  const Inner<kSteps> inner(a, tile, rank, row);
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
    } else if constexpr (kWidth != kNarrow) {
      x.base = load_quad(a.residual + at, n + 4 * g, width, kWidth == kRagged && n + 16 > width);
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
    if constexpr (kWidth != kNarrow) {
      store_quad<false>(a.out + at, n + 4 * g, width, kWidth == kRagged, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + 4 * g + i < last)
          a.out[at + n + 4 * g + i] = v[i];
    }
  };
  for (; n0 < last; n0 += kAhead * stride) {
    Columns x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (n0 + u * stride < last)
        load(n0 + u * stride, x[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (n0 + u * stride < last)
        finish(n0 + u * stride, x[u]);
  }
}

// Tiles of more than 16 rows: a block takes 128 columns at a time, a wave 16 rows of them
// (4096 prompt rows 141 us against 178 from registers in rows of 64 bytes, where 16
// neighbouring lanes write 16 rows; 127 -> 116 with stores that pass the cache by, as the
// outputs are not read here again).
// The columns' weights pass through LDS for the four waves, the next ones on their way
// meanwhile; so do a wave's products, which it adds to the residual in whole runs of 512
// bytes of a row.
constexpr int kWide = 128;
template <int kSteps> struct WideShared {
  // (16 bytes more a row: neighbouring rows start on other banks.)
  __attribute__((aligned(16))) uint16_t weight[kWide][32 * kSteps + 8];
  __attribute__((aligned(16))) float product[kTileRows][kWide + 4];
};
template <int kSteps, int kWidth, bool kResidual>
__device__ inline void up_wide(const AdapterArgs &a, const TileRows &list, int begin, int last,
                               WideShared<kSteps> &shared) {
  const Tile &tile = list.tile;
  constexpr int kPieces = kWide * 4 * kSteps / 256;  // 16 bytes of weights a thread
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int width = a.pool.out_width, rank = rank_of(a.pool, tile.adapter);
  const uint16_t *up = a.pool.up + tile.adapter * a.pool.up_stride;
  const int row = list.list[min(16 * wave + col, tile.count - 1)];
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
  const Inner<kSteps> inner(a, tile, rank, row);
  const RankMask<kSteps> mask(rank);
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
        base[i] = load_quad(a.residual + at[i], n, width, kWidth == kRagged && n0 + kWide > width);
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
      if (t < rows)
        store_quad<true>(a.out + at[i], n, width, kWidth == kRagged, base[i] + v);
    }
    wave_sync();
  }
}

template <int kSteps, int kWidth, bool kResidual>
__global__ __launch_bounds__(256) void up_kernel(const AdapterArgs a) {
  extern __shared__ f32x4 up_shared[];  // WideShared, if any tile goes through it
  __shared__ TileRows rows;
  int chunk = a.chunk, chunks = (a.pool.out_width + chunk - 1) / chunk;
  if (a.narrow) {
    // Narrower chunks by the tiles that there are, but two units where inner values cost more,
    // unless that leaves CUs without a block. (The tile is loaded meanwhile.)
    Tile own{-1, 0, 0, 0};
    if (static_cast<int>(threadIdx.x) < a.tiles)
      own = a.tile[threadIdx.x];
    const int found = max(1, min(*a.found, a.tiles)), unit = kWide;
    const int units = (a.pool.out_width + unit - 1) / unit;
    const int enough = max(kSteps > 1 ? (units + 1) / 2 : units, kCus / found);
    const int more = max(1, min(static_cast<int>(gridDim.x) / found, min(units, enough)));
    chunk = (units + more - 1) / more * unit;
    chunks = (a.pool.out_width + chunk - 1) / chunk;
    const int index = static_cast<int>(blockIdx.x) / chunks;
    if (index >= found)
      return;
    if (static_cast<int>(threadIdx.x) == index)
      rows.tile = checked_tile(a, own);
    __syncthreads();
    find_rows(a, rows.tile, rows);
    __syncthreads();
  } else {
    find_tile(a, static_cast<int>(blockIdx.x) / chunks, rows);
  }
  const Tile tile = rows.tile;
  if (tile.count == 0)
    return;
  const int begin = static_cast<int>(blockIdx.x) % chunks * chunk;
  const int last = min(a.pool.out_width, begin + chunk);
  if (tile.adapter < 0) {
    if (a.residual != a.out)
      copy_rows<kResidual>(a, rows, begin, last);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (kWidth != kNarrow) {
    if (tile.count > 16 && a.wide) {
      up_wide<kSteps, kWidth, kResidual>(
          a, rows, begin, last, *reinterpret_cast<WideShared<kSteps> *>(up_shared));
      return;
    }
  }
  const int sets = tile.count <= 16 ? 1 : tile.count <= 32 ? 2 : 4;
  if (16 * (wave % sets) < tile.count)
    up_rows<kSteps, kWidth, kResidual>(a, rows, wave % sets, begin + 16 * (wave / sets),
                                       64 / sets, last);
}

// ------------------------------------------------------------- little work
// Both products of a row in one launch, which waits for nothing but the row's adapter: each
// block forms all inner values of its row again, and some columns. A wave takes 8 ranks and
// 512 of the width, whole runs of 1 KB; kLanes neighbouring lanes share a column, 8 ranks
// each. One row of rank 16, width 4096 -> 12288, takes 6.6 us, two launches 8.9; 96 rows of 40
// adapters 14.1 and 18.7. Bound by L2, from which every block reads its adapter, and up to
// rank 32 by as many instructions; above, matrix instructions form the inner values, which cost
// 1 us more to begin with (rank 8 6.5 and 7.8 us; rank 128, width 1920, 13.3 and 11.4).
constexpr int kBothThreads = 1024, kSliceWidth = 512;
// Values of an adapter's down that this pays for at most.
constexpr size_t both_weights(int rank) { return rank <= 32 ? 1 << 17 : (1 << 18) - 1; }
constexpr int kBothSums = static_cast<int>(both_weights(32) / (8 * kSliceWidth)) + 32 / 8;
static_assert(kBothSums >= kBothThreads / 64 && kMostRank / 8 <= kBothThreads / 64,
              "all partial sums have a place, each 8 ranks a wave");
template <int kLanes> __device__ inline float lanes_sum(float v) {
  if constexpr (kLanes > 1)
    v += dpp<0xb1, 0xf>(v, v);  // quad_perm 1 0 3 2
  if constexpr (kLanes > 2)
    v += dpp<0x4e, 0xf>(v, v);  // quad_perm 2 3 0 1
  if constexpr (kLanes > 4)
    v += dpp<0x141, 0xf>(v, v);  // row_half_mirror
  if constexpr (kLanes > 8)
    v += dpp<0x140, 0xf>(v, v);  // row_mirror
  return v;
}
template <int kLanes, bool kLow, bool kResidual>
__global__ __launch_bounds__(kBothThreads) void both_kernel(const AdapterArgs a) {
  __shared__ __attribute__((aligned(16))) float partial[kBothSums][8], inner[kMostRank];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int out_width = a.pool.out_width, width = a.pool.in_width;
  const int chunks = (out_width + a.chunk - 1) / a.chunk;
  const int row = static_cast<int>(blockIdx.x / chunks);
  const int begin = static_cast<int>(blockIdx.x % chunks) * a.chunk;
  const int last = min(out_width, begin + a.chunk);
  const size_t at = row * a.out_stride;
  const int adapter = checked_adapter(a, row);
  if (adapter == a.pool.adapters) {
    if (a.residual != a.out)
      for (int n = begin + threadIdx.x; n < last; n += kBothThreads)
        a.out[at + n] = kResidual ? a.residual[at + n] : 0.0F;
    return;
  }
  const int rank = rank_of(a.pool, adapter);
  const uint16_t *down = a.pool.down + adapter * a.pool.down_stride;
  const uint16_t *up = a.pool.up + adapter * a.pool.up_stride;

  // The first columns' operands are on their way with the inner values'.
  constexpr int kColumns = kBothThreads / kLanes;
  const int k = 8 * (threadIdx.x % kLanes);
  int n0 = begin, n = begin + static_cast<int>(threadIdx.x) / kLanes;
  bf16x8 weight;
  float base = 0.0F;
  const auto request = [&]() {
    const size_t column = min(n, out_width - 1);
    weight = load8(up + column * a.pool.rank + (k < a.pool.rank ? k : 0));
    if constexpr (kResidual)
      base = a.residual[at + column];
  };
  request();

  constexpr int kWaves = kBothThreads / 64;
  const int groups = (rank + 7) / 8;
  int sums;  // of a group
  if constexpr (kLanes <= 4) {
    sums = (width + kSliceWidth - 1) / kSliceWidth;
    for (int unit = wave; unit < groups * sums; unit += kWaves) {
      const int from = unit / groups * kSliceWidth + 8 * lane, first = unit % groups * 8;
      const int where = from < width ? from : 0;
      bf16x8 w[8], low{};
      const bf16x8 high = load8(a.hi + row * a.x_stride + where);
      if constexpr (kLow)
        low = load8(a.lo + row * a.x_stride + where);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        w[r] = load8(down + static_cast<size_t>(min(first + r, rank - 1)) * width + where);
      asm volatile("" ::: "memory");
      float sum[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        sum[r] = 0.0F;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float value = static_cast<float>(w[r][e]);
          sum[r] = fmaf(value, static_cast<float>(high[e]), sum[r]);
          if constexpr (kLow)
            sum[r] = fmaf(value, static_cast<float>(low[e]), sum[r]);
        }
        sum[r] = wave_reduce(from < width ? sum[r] : 0.0F, Sum());
      }
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          partial[unit][r] = sum[r];
      }
    }
  } else {
    // The same runs as both operands of a matrix product: what element i of its diagonal
    // sums up are lanes i, i + 16, .. of both. A wave takes every `sums`th slice.
    sums = max(1, kWaves / max(1, groups));
    if (wave < groups * sums) {
      const int first = wave % groups * 8;
      f32x4 sum[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        sum[r] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
      for (int slice = wave / groups * kSliceWidth; slice < width; slice += sums * kSliceWidth) {
        const int from = slice + 8 * lane, where = from < width ? from : 0;
        bf16x8 w[8], low{}, high = load8(a.hi + row * a.x_stride + where);
        if constexpr (kLow)
          low = load8(a.lo + row * a.x_stride + where);
#pragma unroll
        for (int r = 0; r < 8; ++r)
          w[r] = load8(down + static_cast<size_t>(min(first + r, rank - 1)) * width + where);
        asm volatile("" ::: "memory");
        if (slice + kSliceWidth > width && from >= width) {
          high = low = bf16x8{};
#pragma unroll
          for (int r = 0; r < 8; ++r)
            w[r] = bf16x8{};
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r], high, sum[r], 0, 0, 0);
          if constexpr (kLow)
            sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r], low, sum[r], 0, 0, 0);
        }
      }
      const bool diagonal = lane >> 4 == (lane & 15) >> 2;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float even = (lane & 2) != 0 ? sum[r][2] : sum[r][0];
        const float odd = (lane & 2) != 0 ? sum[r][3] : sum[r][1];
        const float own = (lane & 1) != 0 ? odd : even;
        const float all = wave_reduce(diagonal ? own : 0.0F, Sum());
        if (lane == 0)
          partial[wave][r] = all;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < kMostRank) {
    const int r = threadIdx.x;
    float v = 0.0F;
    if (r < rank) {
      for (int i = 0; i < sums; ++i)
        v += partial[i * groups + r / 8][r % 8];
      v *= a.pool.scales == nullptr ? 1.0F : a.pool.scales[adapter];
    }
    inner[r] = v;
  }
  __syncthreads();
  float values[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    values[e] = inner[k + e];
  for (;;) {
    float v = 0.0F;
#pragma unroll
    for (int e = 0; e < 8; ++e)  // (Behind the rank the weights may be anything.)
      v = k + e < rank ? fmaf(static_cast<float>(weight[e]), values[e], v) : v;
    v = lanes_sum<kLanes>(v);
    if (k == 0 && n < last)
      a.out[at + n] = base + v;
    n0 += kColumns;
    n += kColumns;
    if (n0 >= last)
      break;
    request();
  }
}

// ---------------------------------------------------------------------- host
// Tiles at most: each bin's last tile may be short.
size_t most_tiles(const AdapterPool &pool, size_t rows) {
  if (rows <= kSingleRows)
    return rows;
  return std::min(rows, rows / kTileRows + std::min<size_t>(rows, pool.adapters + size_t{1}));
}
// 32s of ranks in the second product.
int steps_of(const AdapterPool &pool) { return pool.rank <= 32 ? 1 : pool.rank <= 64 ? 2 : 4; }
// From kManyRows on their own tiles outweigh those that adapters add, so the tiles that there
// usually are (the adapters' last ones half as many) say how full the card is.
size_t usual_tiles(const AdapterPool &pool, size_t rows) {
  return std::min(most_tiles(pool, rows),
                  rows / kTileRows + std::min<size_t>(rows, pool.adapters + size_t{1}) / 2 + 1);
}
// Whether tiles are expected to have more than 16 rows: most_tiles is about twice what
// rows of a few adapters fill. (Tiles of 16 rows and fewer are formed from registers: their
// lanes write whole 64 bytes of few rows.)
bool wide_tiles(const AdapterPool &pool, size_t rows) {
  return rows > 8 * most_tiles(pool, rows);
}
// Blocks for a tile's rows: two where many tiles have more than 32, or there are few rows.
// (8192 rows of 8000 adapters 157 us, now 134; 1000 rows of 1000 131 and 113.)
size_t halves_of(const AdapterPool &pool, size_t rows) {
  return rows <= 32 || (rows > kFewRows && !wide_tiles(pool, rows)) ? 1 : 2;
}
// 16s of ranks in a block of down_kernel at most.
int ranks_of(const AdapterPool &pool, size_t rows) {
  return pool.rank <= 16 ? 1 : pool.rank <= 32 ? 2 : pool.rank <= 64 || rows <= kFewRows ? 4 : 8;
}
// Blocks of down_kernel. Two fit a CU, but where a block takes 128 ranks (above rank 64, with
// more than kFewRows rows), 128 KB of LDS and 160 registers, one.
size_t down_blocks(const AdapterPool &pool, size_t rows, size_t parts) {
  const size_t units = most_tiles(pool, rows) * halves_of(pool, rows) *
                       ceil_div(pool.rank, 16 * ranks_of(pool, rows));
  return rows <= kFewRows ? std::max<size_t>(units, 512) : units * parts;
}
// Parts of the width at most: about four steps a wave (two up to rank 32, whose parts are
// cheap to add up: 94 rows of rank 96 lose 4 us), but no more than eight, as the second
// product adds them up (width 11264, us with 8, 6 and 4: 220 rows of rank 40 17.8, 21.0 and
// 22.3, 109 rows of rank 24 15.1, 16.6 and 18.2). The kernel takes fewer, by the tiles that it
// finds. Above kFewRows they are chosen here: as many as make 512 blocks if the tiles
// are its most; for many rows so that the busiest CU has least to do, its
// blocks' steps and about 8 more for each, and for a part what the second product does with it.
// (512 blocks of 128 ranks may take two rounds. us with 512 and 256 of them, 12 adapters of
// rank 128, width 11264: 513 rows 35.0 and 39.5, 700 rows 36.4 and 42.5, 1000 rows 56.2 and
// 48.3, 1500 rows 84.7 and 72.4; 2047 rows of 4, width 4096, 72.6 and 75.0. Rank 72 is alike.)
size_t parts_of(const AdapterPool &pool, size_t rows) {
  const size_t steps = (static_cast<size_t>(pool.in_width) + 31) / 32;
  const size_t parts = std::min<size_t>(8, ceil_div(steps, 4 * kDownWaves));
  if (rows <= kFewRows)
    return pool.rank <= 32 ? std::min<size_t>(8, ceil_div(steps, 2 * kDownWaves)) : parts;
  const size_t halves = halves_of(pool, rows);
  if (rows < kManyRows)
    return std::max<size_t>(1, std::min(parts, 512 / (halves * most_tiles(pool, rows))));
  const size_t units = usual_tiles(pool, rows) * halves;
  size_t best = 1, least = ~size_t{0};
  for (size_t p = 1; p <= parts; ++p) {
    const size_t cost =
        ceil_div(units * p, kCus) * (ceil_div(steps, p) + 8) + 4 * p * steps_of(pool);
    if (cost < least)
      best = p, least = cost;
  }
  return best;
}
// Whether group_kernel sorts: many rows, or many blocks that would each sort them (us with and
// without its launch: 4096 prompt rows on 8 adapters, 438 blocks, 113.1 and 110.2, 513 rows of
// 4 19.1 and 16.9; 4000 rows of 2000 adapters, 2062 blocks, 193 and 218).
bool sorted_first(const AdapterPool &pool, size_t rows) {
  return rows > kSelfRows ||
         (rows > kFewRows && down_blocks(pool, rows, parts_of(pool, rows)) > kMostSorts);
}
// Output columns of a block: few blocks, as each forms its tile's inner values again: 512 with
// LDS, 2048 without. (Two with LDS fit a CU at once, up to rank 64 mostly three. us with 512
// and 768 blocks: 513 rows of 4 adapters of rank 16 20.3 and 19.9, 512 of 6 of rank 64 23.9 and
// 23.5, but 2047 of 4 of rank 64 59.5 and 61.7, and of 7, width 11264 -> 4096, 57.2 and 54.4,
// 1000 of them 27.2 and 29.0.) With many rows 512 would
// leave some CUs one block and others two, so there the busiest CU has least to do, in
// quarters of 128 columns, of which inner values cost a block two for each 32 ranks (with the
// parts above, width 4096, rank 16: 16384 rows 207 us for 261, 8192 rows 96 for 107, 4096 rows
// of 256 adapters 67 for 83).
size_t chunk_of(const AdapterPool &pool, size_t rows, bool wide) {
  const size_t width = static_cast<size_t>(pool.out_width), unit = wide ? kWide : 64;
  const size_t units = ceil_div(width, unit), fit = (wide ? 512 : 2048) / most_tiles(pool, rows);
  size_t chunks = std::max<size_t>(1, std::min(units, fit));
  if (wide && rows >= kManyRows) {
    size_t least = ~size_t{0};
    for (size_t c = 1; c <= std::min<size_t>(units, 16); ++c) {
      const size_t cost = ceil_div(usual_tiles(pool, rows) * c, kCus) *
                          (4 * ceil_div(units, c) + 2 * steps_of(pool));
      if (cost < least)
        chunks = c, least = cost;
    }
  }
  return ceil_div(ceil_div(width, chunks), unit) * unit;
}
// Whether up_kernel divides its columns by the tiles found, which costs 0.3 us: for pools of
// which a batch may use few (us without and with, width 4096 -> 12288, 3 of 20 adapters: 200
// rows of rank 16 19.0 and 15.9, 1600 rows of rank 64 56.7 and 46.2; all 4 of 4: 18.7 and 19.0).
bool narrow_chunks(const AdapterPool &pool, size_t rows) {
  return wide_tiles(pool, rows) && rows < kManyRows && pool.adapters >= 8 &&
         most_tiles(pool, rows) <= 256;
}
size_t order_of(const AdapterPool &pool, size_t rows) {
  return !sorted_first(pool, rows) ? most_tiles(pool, rows) * kTileRows : rows;
}
size_t aligned(size_t bytes) { return (bytes + 15) / 16 * 16; }

// Whether both_kernel takes the call: where an adapter is read in 3 us, and all rows' work takes
// no longer than a launch. us of both_kernel and of tiles: width 4096 -> 12288, 128 rows of
// rank 16 11.6 and 14.8, 192 rows 17.7 and 15.3; 64 rows of rank 32 13.4 and 15.0, 96 rows
// 19.1 and 15.3; 16 rows of rank 48 13.0 and 17.5; one row of rank 64 12.4 and 11.3, of rank 32
// and width 11264 13.9 and 11.2; width 1920 -> 5760, 32 rows of rank 128 18.6 and 20.3.
bool both_at_once(const AdapterPool &pool, size_t rows) {
  const size_t rank = static_cast<size_t>(pool.rank), width = static_cast<size_t>(pool.in_width);
  return rows <= kFewRows && rank * width <= both_weights(pool.rank) &&
         rows * rank * (width + pool.out_width) <= size_t{1} << 25;
}
template <int kLanes> Status launch_both(AdapterArgs a, hipStream_t stream) {
  const size_t width = static_cast<size_t>(a.pool.out_width);
  // (Twice as many blocks than CUs take 1 to 3 us more.)
  const size_t chunks = std::max<size_t>(1, kCus / a.rows);
  a.chunk = static_cast<int>(ceil_div(ceil_div(width, chunks), 16) * 16);
  const size_t blocks = a.rows * ceil_div(width, a.chunk);
  const auto choose = [&](auto low) {
    constexpr bool kLow = decltype(low)::value;
    return a.residual != nullptr ? both_kernel<kLanes, kLow, true>
                                 : both_kernel<kLanes, kLow, false>;
  };
  const auto kernel = a.lo != nullptr ? choose(std::true_type()) : choose(std::false_type());
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBothThreads), 0, stream,
                     a);
  return launch_status("adapter both_kernel");
}
template <int kRanks>
Status launch_down(const AdapterArgs &a, size_t blocks, hipStream_t stream) {
  const auto kernel = a.lo != nullptr ? down_kernel<kRanks, true> : down_kernel<kRanks, false>;
  const int cols = a.rows <= 16 ? 1 : 2;  // 16s of rows in a block
  const int loads = kRanks + cols * (a.lo != nullptr ? 2 : 1);
  const size_t bins = a.sorted ? 0 : (a.pool.adapters + 1) * sizeof(int32_t);
  const size_t lds =
      std::max(bins, kDownWaves * std::max(loads, kRanks * cols) * 64 * sizeof(f32x4));
  if (lds > 64 * 1024)
    EVO_TRY(hip_status(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)),
                       "adapter down_kernel LDS opt-in"));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)),
                     dim3(64 * kDownWaves), static_cast<unsigned>(lds), stream, a);
  return launch_status("adapter down_kernel");
}
template <int kSteps>
Status launch_up(const AdapterArgs &a, size_t chunks, hipStream_t stream) {
  const auto choose = [&](auto width) {
    constexpr int kWidth = decltype(width)::value;
    return a.residual != nullptr ? up_kernel<kSteps, kWidth, true>
                                 : up_kernel<kSteps, kWidth, false>;
  };
  const bool quads = a.pool.out_width >= 4;
  const auto kernel = !quads                      ? choose(std::integral_constant<int, kNarrow>{})
                      : a.pool.out_width % 4 == 0 ? choose(std::integral_constant<int, kWhole>{})
                                                  : choose(std::integral_constant<int, kRagged>{});
  const size_t lds = quads && a.wide ? sizeof(WideShared<kSteps>) : 0;
  if (lds > 64 * 1024)
    EVO_TRY(hip_status(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)),
                       "adapter up_kernel LDS opt-in"));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.tiles * chunks)), dim3(256),
                     static_cast<unsigned>(lds), stream, a);
  return launch_status("adapter up_kernel");
}

Status invalid(const char *why) { return {ErrorCode::kInvalidArgument, why}; }

}  // namespace

// What a call uses: the rows' bins, their order, the tiles, how many there are, inner values.
size_t adapter_workspace_used(const AdapterPool &pool, size_t rows) {
  return aligned(rows * sizeof(int32_t)) + aligned(order_of(pool, rows) * sizeof(int32_t)) +
         aligned(most_tiles(pool, rows) * sizeof(Tile)) + 16 +
         parts_of(pool, rows) * rows * pool.rank * sizeof(float);
}
// That falls where more rows take fewer parts or another sort; this bounds it for `rows` and
// all fewer. Its terms, for r <= rows: tiles grow with r but from 4 rows on to 5; the order
// holds r, or 64 for each tile up to kSelfRows. Parts times r is at most `few` r up to
// kFewRows and `many` r above; and never more than r + 2048 (steps + 8): below kManyRows as
// parts are steps / 16 + 1 at most, from there on as the model of parts_of takes p > 1 only if
// units / 256 * 8 (p - 1) < steps + 8, and units exceed r / 64 - 1.
size_t adapter_workspace_bytes(const AdapterPool &pool, size_t rows) {
  const auto tiles = [&](size_t r) {
    return std::max(most_tiles(pool, r), std::min<size_t>(r, kSingleRows));
  };
  const size_t order = std::max(rows, tiles(std::min<size_t>(rows, kSelfRows)) * kTileRows);
  const size_t steps = (static_cast<size_t>(pool.in_width) + 31) / 32;
  const size_t few = std::min<size_t>(8, ceil_div(steps, 2 * kDownWaves));
  const size_t many = std::min<size_t>(8, ceil_div(steps, 4 * kDownWaves));
  const size_t inner = std::min(std::max(few * std::min<size_t>(rows, kFewRows), many * rows),
                                rows + 2048 * (steps + 8));
  return aligned(rows * sizeof(int32_t)) + aligned(order * sizeof(int32_t)) +
         aligned(tiles(rows) * sizeof(Tile)) + 16 + inner * pool.rank * sizeof(float);
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
      workspace_bytes < adapter_workspace_used(pool, rows))
    return invalid("adapter_linear: workspace too small or not aligned");
  const size_t tiles = most_tiles(pool, rows), parts = parts_of(pool, rows);
  const bool wide = wide_tiles(pool, rows);
  const size_t width = static_cast<size_t>(pool.out_width), chunk = chunk_of(pool, rows, wide);
  // (2^20 rows are 24577 tiles at most, so both grids are far from 2^32 threads.)
  const size_t chunks = ceil_div(width, chunk);
  const size_t blocks = down_blocks(pool, rows, parts);
  char *const base = static_cast<char *>(workspace);
  const size_t list = aligned(rows * sizeof(int32_t));
  char *const after = base + list + aligned(order_of(pool, rows) * sizeof(int32_t));
  const AdapterArgs args{pool, adapter, x_hi, x_lo, x_stride, static_cast<int>(rows), residual,
                         out, out_stride, static_cast<int>(tiles), static_cast<int>(parts),
                         static_cast<int>(chunk), sorted_first(pool, rows) ? 1 : 0,
                         static_cast<int>(halves_of(pool, rows)), wide ? 1 : 0,
                         narrow_chunks(pool, rows) ? 1 : 0,
                         reinterpret_cast<int32_t *>(base),
                         reinterpret_cast<int32_t *>(base + list),
                         static_cast<int>(order_of(pool, rows)), reinterpret_cast<Tile *>(after),
                         reinterpret_cast<int32_t *>(after + aligned(tiles * sizeof(Tile))),
                         reinterpret_cast<float *>(after + aligned(tiles * sizeof(Tile)) + 16)};
  if (both_at_once(pool, rows))
    return pool.rank <= 8    ? launch_both<1>(args, stream)
           : pool.rank <= 16 ? launch_both<2>(args, stream)
           : pool.rank <= 32 ? launch_both<4>(args, stream)
           : pool.rank <= 64 ? launch_both<8>(args, stream)
                             : launch_both<16>(args, stream);
  if (args.sorted)
    hipLaunchKernelGGL(group_kernel, dim3(1), dim3(rows <= 1024 ? 256 : kGroupThreads),
                       static_cast<unsigned>((pool.adapters + 1) * sizeof(int32_t)), stream,
                       args);
  const int ranks = ranks_of(pool, rows);
  EVO_TRY(ranks == 1   ? launch_down<1>(args, blocks, stream)
          : ranks == 2 ? launch_down<2>(args, blocks, stream)
          : ranks == 4 ? launch_down<4>(args, blocks, stream)
                       : launch_down<8>(args, blocks, stream));
  return pool.rank <= 32   ? launch_up<1>(args, chunks, stream)
         : pool.rank <= 64 ? launch_up<2>(args, chunks, stream)
                           : launch_up<4>(args, chunks, stream);
}

}  // namespace evo::hip
