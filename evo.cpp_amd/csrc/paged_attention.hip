// SPDX-License-Identifier: Apache-2.0
// Attention of a batch's rows over the paged cache: out = sum_k p_k v_k with
// p = softmax(scale q.k) over a row's keys 0 .. position, grouped heads, and
// optionally a prefix that the whole batch shares and that is read once.
//
// The rows of one key/value head are its tokens times the group of query heads
// that read it, side by side: a sequence's rows meet its own keys, and the
// rows of the whole batch meet the shared keys. Each block takes a tile of rows
// and a chunk of keys; a row whose keys lie in several chunks leaves (running
// maximum, sum, unnormalised output) per chunk in the workspace, F32, joined
// by paged_combine_kernel in chunk order.
//
// Products run on v_mfma_f32_16x16x32 as S^T = K Q^T and O^T = V^T P^T, so a
// lane owns one row (column lane % 16) and its softmax state, and P^T is already
// the second product's operand: with g = lane / 16, S^T leaves the lane keys
// 4g + i and 16 + 4g + i of a 32-key step, and the sum over keys may take them in
// that order as long as V does. K and V go from memory to registers without LDS:
// a K operand is 16 bytes of a key's row as it lies, and a lane loads 8 keys x 8
// elements of V and transposes them with v_perm (one per output word).
// Scores, maxima, sums and outputs are F32; the weights (at most 2^8 before the maximum
// follows, in FP16 2^15) are rounded to the cache's type for the second product, and
// the sum is taken of the rounded ones, so that the weights applied add up to one.
//
// 16 rows a block (one query's group of heads) are bound by the bytes of keys and
// values: 64 sequences of up to 8190 positions, 8 key/value heads of 128, 644 MB, take
// 126 us, 5.1 TB/s, and 5.3 to join their parts. 128 rows a block are bound by issue:
// 4096 tokens on 12288 cached ones, 32 heads over 8, 962 GFLOP, take 905 to 967 us (by
// card), 1.06 to 0.99 PFLOP/s, the matrix cores busy 51% of the cycles and the vector
// units 44%, at the 1.76 GHz that the card's power leaves; an 8192-cubed product of the
// library reaches 1.22 PFLOP/s. Rows of up to 16 take the first form (us with it and with
// the second: 64 sequences of 2000, one token 49 and 56, four tokens 50 and 65; 32
// sequences of 16 tokens, one head a key/value head, 94 and 108).
#include "common.hpp"
#include "ops.hpp"
#include "paged.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace evo::hip {

namespace {

struct AttendArgs {
  PagedCache cache;
  PagedBatch batch;
  const uint16_t *query;
  size_t query_stride;
  uint16_t *out;
  size_t out_stride;
  int heads, group;   // query heads, and how many share a key/value head
  float scale2;       // log2(e) * scale
  int chunk;          // own keys per chunk (a multiple of 64)
  int prefix_chunk;   // shared keys per chunk
  int prefix_slots;   // chunks of the shared keys
  int slots;          // chunks of a row at most, the shared ones first
  int direct;         // a row tile is a sequence
  float *part;        // [tokens][heads][slots][head_dim], unnormalised outputs
  float2 *state;      // [tokens][heads][slots] (maximum, sum)
};

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  typedef bf16x8 vec;
  static __device__ inline f32x4 run(const vec &a, const vec &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ inline f32x16 run(const vec &a, const vec &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // sum + the eight elements.
  static __device__ inline float add(const vec &p, float sum) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair one = {static_cast<__bf16>(1.0F), static_cast<__bf16>(1.0F)};
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 0, 1), one, sum, false);
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 2, 3), one, sum, false);
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 4, 5), one, sum, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(p, p, 6, 7), one, sum, false);
  }
};
template <> struct Mfma<_Float16> {
  typedef f16x8 vec;
  static __device__ inline f32x4 run(const vec &a, const vec &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ inline f32x16 run(const vec &a, const vec &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ inline float add(const vec &p, float sum) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    const pair one = {static_cast<_Float16>(1.0F), static_cast<_Float16>(1.0F)};
    sum = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 0, 1), one, sum, false);
    sum = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 2, 3), one, sum, false);
    sum = __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 4, 5), one, sum, false);
    return __builtin_amdgcn_fdot2(__builtin_shufflevector(p, p, 6, 7), one, sum, false);
  }
};

template <typename T> __device__ inline uint16_t bits_of(float v) {
  return __builtin_bit_cast(uint16_t, static_cast<T>(v));
}

// Chunks of own keys of a row at `position` (-1 and below: it sees nothing).
__device__ inline int own_chunks(const AttendArgs &a, int position) {
  const int keys = position + 1 - a.batch.shared_length;
  return keys <= 0 ? 0 : (keys + a.chunk - 1) / a.chunk;
}
// Whether a row is finished by the block of its first chunk, not joined: it has
// no other.
__device__ inline bool single_chunk(const AttendArgs &a, int position) {
  return a.prefix_slots == 0 && position < a.chunk;
}

// Row tile `tile` of the batch's own-key phase: the tiles of its sequences in
// order, ceil(count * group / kRows) each. Every lane of the wave calls.
template <int kRows>
__device__ inline bool find_tile(const AttendArgs &a, int tile, int *sequence, int *tile_in) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < a.batch.sequences; s0 += 64) {
    int tiles = 0;
    if (s0 + lane < a.batch.sequences) {
      const SequenceRows rows = sequence_rows(a.batch, s0 + lane);
      if (rows.valid)
        tiles = (rows.count * a.group + kRows - 1) / kRows;
    }
    int through = tiles;
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
      const int below = __shfl_up(through, offset, 64);
      through += lane >= offset ? below : 0;
    }
    const uint64_t found = __ballot(base + through > tile);
    if (found != 0) {
      // A sequence's last tiles, which see the most keys, come first.
      const int at = __builtin_ctzll(found);
      *sequence = s0 + at;
      *tile_in = base + __shfl(through, at, 64) - 1 - tile;
      return true;
    }
    base += __shfl(through, 63, 64);
  }
  return false;
}

// The rows a block works on: rows row0 .. of `rows` (a sequence's, or with
// `prefix` the batch's), row r being token first_token + r / group; the positions
// of the tile's first and last row (prefix: the last shared one, which all see).
struct RowTile {
  int sequence, row0, rows, first_token, first_position, last_position;
};
template <int kRows>
__device__ inline bool row_tile(const AttendArgs &a, bool prefix, int tile, RowTile *t) {
  if (prefix) {
    *t = {0, tile * kRows, a.batch.tokens * a.group, 0, a.batch.shared_length - 1,
          a.batch.shared_length - 1};
    return true;
  }
  int sequence = tile, tile_in = 0;
  if (!a.direct && !find_tile<kRows>(a, tile, &sequence, &tile_in))
    return false;
  sequence = __builtin_amdgcn_readfirstlane(sequence);
  const SequenceRows own = sequence_rows(a.batch, sequence);
  if (!own.valid || own.count == 0)
    return false;
  const int row0 = __builtin_amdgcn_readfirstlane(tile_in) * kRows;
  const int rows = own.count * a.group, position = own.length - own.count;
  *t = {sequence, row0, rows, own.first, position + row0 / a.group,
        position + (min(row0 + kRows, rows) - 1) / a.group};
  return true;
}

// Block -> phase, key/value head, chunk and row tile. Heads vary fastest: with a
// multiple of eight of them the blocks of a head share an XCD's L2.
struct BlockWork {
  bool prefix;
  int kv_head, chunk, tile;
};
__device__ inline BlockWork block_work(const AttendArgs &a, unsigned prefix_blocks) {
  BlockWork w;
  w.prefix = blockIdx.x < prefix_blocks;
  unsigned rest = w.prefix ? blockIdx.x : blockIdx.x - prefix_blocks;
  w.kv_head = static_cast<int>(rest % a.cache.kv_heads);
  rest /= a.cache.kv_heads;
  const unsigned chunks = w.prefix ? a.prefix_slots : a.slots - a.prefix_slots;
  w.chunk = static_cast<int>(rest % chunks);
  w.tile = static_cast<int>(rest / chunks);
  return w;
}

// A weight may exceed the running maximum's by 2^kSlack before the maximum follows. The
// wave branches as one, but each row follows by its own scores alone: another base rounds
// its weights differently, and its bits must not depend on what other rows see.
// The maximum's own weight is 2^kLift, in the sum and the outputs alike. FP16 spans few
// powers of two: unlifted, weights below 2^-14 lost bits and those below 2^-25 were
// nothing, all of a row's output where its leading key has small values. Lifted by 9 it
// holds weights down to 2^-23 of the largest in full and every one to 2^-34. The slack
// leaves room below 2^16; less slack and more lift costs prompts (4096 tokens, us: slack
// 2 180, 4 173, 5 167, 6 and 8 165).
template <typename T> constexpr float kSlack = std::is_same_v<T, _Float16> ? 6.0F : 8.0F;
template <typename T> constexpr float kLift = std::is_same_v<T, _Float16> ? 9.0F : 0.0F;

// Weight of a score where that of `base` is 1. The difference is scaled, not the two
// scores: their products' roundings would leave 2^(+-256) of it at scores of 2^32.
__device__ inline float weight(float score, float base, float scale2) {
  return __builtin_amdgcn_exp2f((score - base) * scale2);
}
// The same lifted, for the cache's type T.
template <typename T> __device__ inline float lifted(float score, float base, float scale2) {
  return __builtin_amdgcn_exp2f(fmaf(score - base, scale2, kLift<T>));
}
// 128-row blocks form exp2(score * scale2 - base * scale2) all the same, with one
// instruction less a score (4096 tokens on 12288 cached ones 938 us, else 963), where
// the base's product is below this, so that its rounding is below 2^-14. A row beyond
// has its base taken from its scores first.
constexpr float kNear = 1024.0F;
__device__ inline bool is_far(float top, float scale2) {
  return top != -INFINITY && !(fabsf(top * scale2) < kNear);
}

// Softmax state and output of 16 rows over the keys a wave has seen. Lane l:
// row l % 16, output elements kVec * (4 * (l / 16) + i) + t for i < 4, t < kVec.
template <int kD> struct RowState {
  static constexpr int kVec = kD / 16;
  float top, sum;  // a score as it is; the sum of this lane's own keys
  f32x4 out[kVec];
};

// One 32-key step. k[u][s]: K operand of keys 16u .., elements 32s ..; v[j]: this
// lane's 8 keys, kD / 16 elements each.
template <typename T, int kD> struct Step {
  typename Mfma<T>::vec k[2][kD / 32];
  uint32_t v[8][kD / 32];
};

template <int kWords>
__device__ inline void load_words(const uint16_t *src, uint32_t (&w)[kWords]) {
  if constexpr (kWords == 4) {
    const uint4 q = *reinterpret_cast<const uint4 *>(src);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  } else if constexpr (kWords == 2) {
    const uint2 q = *reinterpret_cast<const uint2 *>(src);
    w[0] = q.x, w[1] = q.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(src);
  }
}

// K and V of 16 keys from k0 (a multiple of 16) in page `page`: the keys share it.
template <typename T, int kD>
__device__ inline void load_keys(const AttendArgs &a, int kv_head, int k0, int page,
                                 typename Mfma<T>::vec (&k)[kD / 32]) {
  const int lane = threadIdx.x & 63;
  const uint16_t *base = a.cache.keys + (page * a.cache.page_stride +
                                         kv_head * a.cache.head_stride +
                                         (k0 & ((1 << a.cache.page_shift) - 1)) *
                                             a.cache.token_stride);
  const uint32_t offset =
      (lane & 15) * static_cast<uint32_t>(a.cache.token_stride) + 8 * (lane >> 4);
#pragma unroll
  for (int s = 0; s < kD / 32; ++s)
    k[s] = *reinterpret_cast<const typename Mfma<T>::vec *>(base + offset + 32 * s);
}
template <int kD>
__device__ inline void load_values(const AttendArgs &a, int kv_head, int k0, int page,
                                   uint32_t (*v)[kD / 32]) {
  const int lane = threadIdx.x & 63;
  const uint16_t *base = a.cache.values + (page * a.cache.page_stride +
                                           kv_head * a.cache.head_stride +
                                           (k0 & ((1 << a.cache.page_shift) - 1)) *
                                               a.cache.token_stride);
  const uint32_t stride = static_cast<uint32_t>(a.cache.token_stride);
  const uint32_t offset = 4 * (lane >> 4) * stride + kD / 16 * (lane & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    load_words(base + offset + i * stride, v[i]);
}

// S^T of a step for 16 rows: entry i of score[u] is key 16u + 4 * (lane / 16) + i.
template <typename T, int kD>
__device__ inline void scores(const Step<T, kD> &step, const typename Mfma<T>::vec *q,
                              f32x4 (&score)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    score[u] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (int s = 0; s < kD / 32; ++s)
      score[u] = Mfma<T>::run(step.k[u][s], q[s], score[u]);
  }
}

// Infinities and NaN in a word of two elements.
template <typename T> __device__ inline bool nonfinite(uint32_t word) {
  constexpr uint32_t kExponent = std::is_same_v<T, __bf16> ? 0x7f80U : 0x7c00U;
  return (word & kExponent) == kExponent || (word >> 16 & kExponent) == kExponent;
}
template <typename T> __device__ inline float element(uint16_t bits) {
  return static_cast<float>(__builtin_bit_cast(T, bits));
}

// Adds a step's scores and values to the rows' state.
template <typename T, int kD>
__device__ inline void attend(const f32x4 (&score)[2], const uint32_t (&v)[8][kD / 32],
                              float scale2, RowState<kD> &state) {
  constexpr int kVec = kD / 16;
  typedef typename Mfma<T>::vec vec;
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = fmaxf(top, score[u][i]);
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const bool follows = (top - state.top) * scale2 > kSlack<T>;
  if (__any(follows)) {
    const float next = follows ? top : state.top;
    const float shrink = follows ? weight(state.top, next, scale2) : 1.0F;
    state.sum *= shrink;
#pragma unroll
    for (int t = 0; t < kVec; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        state.out[t][i] *= shrink;
    state.top = next;
  }
  const float base = state.top == -INFINITY ? 0.0F : state.top;
  vec p;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[4 * u + i] = static_cast<T>(lifted<T>(score[u][i], base, scale2));
  state.sum = Mfma<T>::add(p, state.sum);
#pragma unroll
  for (int t = 0; t < kVec; ++t) {
    // Element t of this lane's kVec of each of its 8 keys.
    uint32_t word[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      word[j] = __builtin_amdgcn_perm(v[2 * j + 1][t / 2], v[2 * j][t / 2],
                                      t % 2 == 0 ? 0x05040100U : 0x07060302U);
    state.out[t] = Mfma<T>::run(__builtin_bit_cast(vec, word), p, state.out[t]);
  }
}

// The keys of a step (bit 16u + 4 * (lane / 16) + i) with an infinity or NaN among
// their values, which are zeroed.
template <typename T, int kD>
__device__ inline uint32_t odd_keys(uint32_t (&v)[8][kD / 32]) {
  const int g = (threadIdx.x & 63) >> 4;
  uint32_t keys = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    bool odd = false;
#pragma unroll
    for (int w = 0; w < kD / 32; ++w)
      odd |= nonfinite<T>(v[j][w]);
    const uint64_t lanes = __ballot(odd);
#pragma unroll
    for (int other = 0; other < 4; ++other)
      keys |= (lanes >> (16 * other) & 0xffff) != 0 ? 1U << (j / 4 * 16 + 4 * other + j % 4) : 0;
    if ((lanes >> (16 * g) & 0xffff) != 0) {
#pragma unroll
      for (int w = 0; w < kD / 32; ++w)
        v[j][w] = 0;
    }
  }
  return keys;
}

// 16 rows of a key/value head and a chunk of their keys per block; its four waves take
// every fourth 32-key step and join their states through LDS. (Eight waves a block
// took longer at every size: one sequence of 512 keys 9.7 us for 8.9, 60 of them 17.4
// for 15.2.)
// Blocks below prefix_blocks take the shared keys, rows of the whole batch.
template <int kD> struct StreamShared {
  float top[4][16], sum[4][16];
  __attribute__((aligned(16))) float out[4][16][kD + 4];
};
template <typename T, int kD>
__device__ inline void stream_block(const AttendArgs &a, const BlockWork &work,
                                    StreamShared<kD> &shared) {
  constexpr int kRows = 16, kVec = kD / 16, kSteps = kD / 32;
  typedef typename Mfma<T>::vec vec;
  auto &top_s = shared.top, &sum_s = shared.sum;
  auto &out_s = shared.out;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool prefix = work.prefix;
  const int kv_head = work.kv_head, chunk = work.chunk;
  const int key0 = prefix ? chunk * a.prefix_chunk : a.batch.shared_length + chunk * a.chunk;
  int k0 = key0 + 32 * wave;
  // The first step's table entries, requested beside the rows' own description
  // where the table's row is known without it.
  const bool early = prefix || a.direct;
  int entries = -1;
  if (early && lane < 2 &&
      k0 + 16 * lane < (prefix ? a.batch.shared_length : a.batch.max_length)) {
    const int32_t *row = prefix ? a.batch.shared_table
                                : a.batch.page_table + work.tile * a.batch.table_stride;
    entries = row[(k0 + 16 * lane) >> a.cache.page_shift];
  }
  RowTile tile;
  if (!row_tile<kRows>(a, prefix, work.tile, &tile))
    return;
  const int row = tile.row0 + col;
  const bool active = row < tile.rows;
  const int token_in = (active ? row : tile.row0) / a.group;
  const int token = tile.first_token + token_in;
  const int head = kv_head * a.group + (active ? row : tile.row0) % a.group;
  const int position =
      prefix ? tile.last_position : tile.first_position + token_in - tile.row0 / a.group;

  // (The first chunk of a sequence without keys goes on: its rows are zero.)
  const int key1 = min(tile.last_position + 1, key0 + (prefix ? a.prefix_chunk : a.chunk));
  if (key0 >= key1 && (prefix || chunk > 0))
    return;

  vec q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    q[s] = *reinterpret_cast<const vec *>(a.query + token * a.query_stride + head * kD + 32 * s +
                                          8 * g);
    if (!active)
      q[s] = vec{};
  }
  RowState<kD> state;
  state.top = -INFINITY;
  state.sum = 0.0F;
#pragma unroll
  for (int t = 0; t < kVec; ++t)
    state.out[t] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};

  const int32_t *table = prefix ? a.batch.shared_table
                                : a.batch.page_table + tile.sequence * a.batch.table_stride;
  // Pages of a step's two 16-key groups in lanes 0 and 1 (-1: none).
  auto entries_at = [&](int k) {
    const int key = k + 16 * lane;
    return lane < 2 && key < key1 ? table[key >> a.cache.page_shift] : -1;
  };
  auto pages_of = [&](int entry, int k) {
    const bool needed = lane < 2 && k + 16 * lane < key1;
    const bool good = needed && entry >= 0 && entry < a.cache.pages;
    if (needed && !good)
      report(a.batch, kBadPage);
    return good ? entry : -1;
  };
  // V of a step is requested before its scores, K of the next one as soon as the
  // scores are done and the page after that with it, so that loads are always in
  // flight with one set of registers. Without a page the loads go to page 0.
  constexpr int kStride = 32 * 4;
  if (k0 < key1) {
    int pages = pages_of(early ? entries : entries_at(k0), k0);
    int page[2] = {__builtin_amdgcn_readlane(pages, 0), __builtin_amdgcn_readlane(pages, 1)};
    Step<T, kD> step;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      load_keys<T, kD>(a, kv_head, k0 + 16 * u, max(page[u], 0), step.k[u]);
    entries = entries_at(k0 + kStride);
    for (;;) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        load_values<kD>(a, kv_head, k0 + 16 * u, max(page[u], 0), step.v + 4 * u);
      f32x4 score[2];
      scores<T, kD>(step, q, score);
      const int here[2] = {page[0], page[1]}, k_here = k0;
      k0 += kStride;
      const bool more = k0 < key1;
      uint32_t apart = 0;  // keys of the step
      if (more) {
        pages = pages_of(entries, k0);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          page[u] = __builtin_amdgcn_readlane(pages, u);
          load_keys<T, kD>(a, kv_head, k0 + 16 * u, max(page[u], 0), step.k[u]);
        }
        entries = entries_at(k0 + kStride);
      }
      if (here[0] < 0 || here[1] < 0 || k_here + 31 > tile.first_position ||
          k_here + 32 > key1) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int from = k_here + 16 * u + 4 * g;
          const int end = here[u] < 0 ? 0 : key1, visible = min(position + 1, end);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            score[u][i] = from + i < visible ? score[u][i] : -INFINITY;
            // Values no row of the tile sees may be anything, and 0 * NaN is NaN.
#pragma unroll
            for (int w = 0; w < kVec / 2; ++w)
              step.v[4 * u + i][w] = from + i < end ? step.v[4 * u + i][w] : 0;
          }
        }
        // An infinity or NaN among the values of a key that some rows of the tile see
        // and others do not: the key's values go through the products as zeros, and
        // to the rows that see it one by one.
        if (tile.first_position != tile.last_position)
          apart = odd_keys<T, kD>(step.v);
      }
      attend<T, kD>(score, step.v, a.scale2, state);
      for (; apart != 0; apart &= apart - 1) {
        const int key = __builtin_ctz(apart), u = key / 16;
        const float base = state.top == -INFINITY ? 0.0F : state.top;
        float s = score[0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j)
          s = 4 * u + key % 4 == j ? score[j / 4][j % 4] : s;
        s = __shfl(s, 16 * (key % 16 / 4) + col, 64);
        const uint16_t *v =
            a.cache.values + (here[u] * a.cache.page_stride + kv_head * a.cache.head_stride +
                              ((k_here + key) & ((1 << a.cache.page_shift) - 1)) *
                                  a.cache.token_stride);
        const float w = lifted<T>(s, base, a.scale2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < kVec; ++t)
            if (s != -INFINITY)
              state.out[t][i] =
                  fmaf(w, element<T>(v[kVec * (4 * g + i) + t]), state.out[t][i]);
      }
      if (!more)
        break;
    }
  }

  // Join the waves: each leaves its rows' maximum, sum and output.
  state.sum += __shfl_xor(state.sum, 16, 64);
  state.sum += __shfl_xor(state.sum, 32, 64);
  if (g == 0) {
    top_s[wave][col] = state.top;
    sum_s[wave][col] = state.sum;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < kVec; ++t)
      out_s[wave][col][kVec * (4 * g + i) + t] = state.out[t][i];
  __syncthreads();
  // Thread: row tid / 16, elements kVec * (tid % 16) ...
  const int r = threadIdx.x >> 4, d = kVec * (threadIdx.x & 15);
  if (tile.row0 + r >= tile.rows)
    return;
  float top = top_s[0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w)
    top = fmaxf(top, top_s[w][r]);
  float total = 0.0F, o[kVec] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float scale = top_s[w][r] == -INFINITY ? 0.0F : weight(top_s[w][r], top, a.scale2);
    total = fmaf(sum_s[w][r], scale, total);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      o[e] = fmaf(out_s[w][r][d + e], scale, o[e]);
  }
  const int out_row = tile.row0 + r;
  const size_t out_token = tile.first_token + out_row / a.group;
  const int out_head = kv_head * a.group + out_row % a.group;
  const int out_position =
      prefix ? tile.last_position
             : tile.first_position + out_row / a.group - tile.row0 / a.group;
  if (!prefix && single_chunk(a, out_position)) {
    if (chunk > 0)
      return;
    // A row without keys is zero.
    const float inverse = total > 0.0F ? 1.0F / total : total == 0.0F ? 0.0F : total;
    uint16_t *dst = a.out + out_token * a.out_stride + out_head * kD + d;
    uint16_t bits[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      bits[e] = bits_of<T>(o[e] * inverse);
    if constexpr (kVec == 8)
      *reinterpret_cast<uint4 *>(dst) = __builtin_bit_cast(uint4, bits);
    else if constexpr (kVec == 4)
      *reinterpret_cast<uint2 *>(dst) = __builtin_bit_cast(uint2, bits);
    else
      *reinterpret_cast<uint32_t *>(dst) = __builtin_bit_cast(uint32_t, bits);
    return;
  }
  if (key0 > out_position)
    return;  // no key of the chunk is the row's, and no one reads its slot
  const size_t slot = (out_token * a.heads + out_head) * a.slots +
                      (prefix ? chunk : a.prefix_slots + chunk);
  if (d == 0)
    a.state[slot] = make_float2(top, total);
  float *dst = a.part + slot * kD + d;
#pragma unroll
  for (int e = 0; e < kVec; e += 2)
    *reinterpret_cast<float2 *>(dst + e) = make_float2(o[e], o[e + 1]);
}

// ------------------------------------------------------------ many rows
// 128 rows of a key/value head, 32 a wave, over tiles of 64 keys: K and V rows
// are copied to LDS by DMA, double buffered, wave w bringing the tile's 16 keys
// 16w .. (one page) of both. S^T = K Q^T on v_mfma_f32_32x32x16: lane l owns row l
// % 32 and, with h = l / 32, keys 8j + 4h + i of each 32. V^T fragments in that
// order come out of V's rows by ds_read_b64_tr_b16, which hands lane c of 16 the
// column c of a block of 4 keys x 16 elements.
// LDS rows are swizzled in 16-byte units: K so that 8 rows read at one unit hit
// distinct banks, V so that 4 rows read at one pair of units do.
template <int kUnits> __device__ inline int swizzle_k(int row, int unit) {
  return unit ^ ((row * kUnits / 16) & (kUnits - 1));
}
template <int kUnits> __device__ inline int swizzle_v(int row, int unit) {
  return unit ^ ((2 * (row * kUnits / 16)) & (kUnits - 1));
}

// Four keys of this lane's column: the 16 lanes of a group give the addresses of 4
// rows of 16 elements, 4 lanes a row.
template <typename Q> __device__ inline Q transposed(const uint16_t *from) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(Q, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(from)));
}

// V^T operands of keys 16kk .. of a tile: keys 16kk + 4 half + (0 .. 3) and 8 more of
// elements 32t + 16 * (lane / 16 % 2) ..
template <typename T, int kD>
__device__ inline void read_values(const uint16_t *v_s, int kk,
                                   typename Mfma<T>::vec (&v)[kD / 32]) {
  constexpr int kUnits = kD / 8;
  typedef T quad __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
  for (int t = 0; t < kD / 32; ++t) {
    quad part[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 16 * kk + 8 * j + 4 * half + (lane & 15) / 4;
      const int d = 32 * t + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
      part[j] = transposed<quad>(v_s + r * kD + 8 * swizzle_v<kUnits>(r, d / 8) + d % 8);
    }
    v[t] = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <typename T, int kD>
__device__ inline void tile_block(const AttendArgs &a, const BlockWork &work,
                                  uint16_t *tile_lds) {  // [2][K, V][plane], odd keys
  constexpr int kRows = 128, kKeys = 64, kUnits = kD / 8;
  constexpr int kSteps = kD / 16, kTiles = kD / 32;   // K-steps of S^T, 32-row tiles of O^T
  constexpr int kPlane = kKeys * kD;                  // elements of K or V in a stage
  constexpr int kOps = kD / 32;                       // DMAs of 16 keys
  constexpr int kOpRows = 512 / kD;                   // keys of a DMA
  typedef typename Mfma<T>::vec vec;

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool prefix = work.prefix;
  RowTile tile;
  if (!row_tile<kRows>(a, prefix, work.tile, &tile))
    return;
  const int row = tile.row0 + 32 * wave + col;
  const bool active = row < tile.rows;
  const int row_in = active ? row : tile.row0;
  const int token_in = row_in / a.group;
  const size_t token = tile.first_token + token_in;
  const int head = work.kv_head * a.group + row_in % a.group;
  const int first_token_in = tile.row0 / a.group;
  const int position =
      prefix ? tile.last_position : tile.first_position + token_in - first_token_in;
  // Lowest and highest position of the wave's rows (wave_rows: it has some).
  const bool wave_rows = tile.row0 + 32 * wave < tile.rows;
  int wave_first = tile.last_position, wave_last = tile.last_position;
  if (!prefix && wave_rows) {
    const int last_row = min(tile.row0 + 32 * wave + 31, tile.rows - 1);
    wave_first = tile.first_position + (tile.row0 + 32 * wave) / a.group - first_token_in;
    wave_last = tile.first_position + last_row / a.group - first_token_in;
  }

  const int key0 = prefix ? work.chunk * a.prefix_chunk
                          : a.batch.shared_length + work.chunk * a.chunk;
  const int key1 = min(tile.last_position + 1, key0 + (prefix ? a.prefix_chunk : a.chunk));
  if (key0 >= key1 && (prefix || work.chunk > 0))
    return;

  const int32_t *table = prefix ? a.batch.shared_table
                                : a.batch.page_table + tile.sequence * a.batch.table_stride;
  // Table entries of the tile's four 16-key groups in lanes 0 .. 3, and their pages
  // (-1: none). An entry is looked at a tile after its load: to wait for it is to wait
  // for every DMA before it.
  auto entries_at = [&](int k0) {
    const int key = k0 + 16 * lane;
    return lane < 4 && key < key1 ? table[key >> a.cache.page_shift] : -1;
  };
  auto pages_of = [&](int entry, int k0) {
    const bool needed = lane < 4 && k0 + 16 * lane < key1;
    const bool good = needed && entry >= 0 && entry < a.cache.pages;
    if (needed && !good)
      report(a.batch, kBadPage);
    return good ? entry : -1;
  };
  const int first_entries = entries_at(key0);
  int entries = entries_at(key0 + kKeys);  // of the next tile

  vec q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    q[s] = *reinterpret_cast<const vec *>(a.query + token * a.query_stride + head * kD + 16 * s +
                                          8 * half);
    if (!active)
      q[s] = vec{};
  }
  f32x16 out[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      out[t][e] = 0.0F;
  float top = -INFINITY, sum = 0.0F;
  float shift = kLift<T>;  // a weight is exp2(score * scale2 + shift)
  bool far_rows = false;   // some of the wave's

  // This lane's source offset inside a DMA, in bytes (K and V: other swizzles).
  uint32_t k_offset[kOps], v_offset[kOps];
#pragma unroll
  for (int i = 0; i < kOps; ++i) {
    const int r = 16 * wave + kOpRows * i + lane / kUnits;
    const uint32_t down = static_cast<uint32_t>((r & 15) * a.cache.token_stride);
    k_offset[i] = 2 * (down + 8 * swizzle_k<kUnits>(r, lane % kUnits));
    v_offset[i] = 2 * (down + 8 * swizzle_v<kUnits>(r, lane % kUnits));
  }
  const unsigned lds = lds_address(tile_lds) + wave * 16 * kD * 2;
  const int slot_mask = (1 << a.cache.page_shift) - 1;
  auto issue = [&](int k0, int stage, int pages) {
    const int page = __builtin_amdgcn_readlane(pages, wave);
    if (page < 0)
      return;
    const size_t at = page * a.cache.page_stride + work.kv_head * a.cache.head_stride +
                      ((k0 + 16 * wave) & slot_mask) * a.cache.token_stride;
    const unsigned to = lds + stage * (4 * kPlane);
#pragma unroll
    for (int i = 0; i < kOps; ++i) {
      dma16_at(a.cache.keys + at, k_offset[i], to + 1024 * i);
      dma16_at(a.cache.values + at, v_offset[i], to + 2 * kPlane + 1024 * i);
    }
  };

  int pages = pages_of(first_entries, key0);
  issue(key0, 0, pages);
  int stage = 0, odd_tiles = 0, odd_first = 0;
  uint16_t *odd_s = tile_lds + 4 * kPlane;  // [tile][wave], 16 keys a bit each
  for (int k0 = key0; k0 < key1; k0 += kKeys, stage ^= 1) {
    wait_dma<0>();
    // Values that no row sees (behind the last key, or of no page) may be
    // anything, and 0 * NaN is NaN: their rows in LDS are zeroed.
    const uint64_t missing = ~__ballot(pages >= 0) & 15;
    if (missing != 0 || k0 + kKeys > key1) {
      const int own = k0 + 16 * wave;
      const int good = (missing >> wave & 1) != 0 ? 0 : min(16, max(0, key1 - own));
      uint16_t *v = tile_lds + stage * 2 * kPlane + kPlane + 16 * wave * kD;
      for (int i = good * kUnits + lane; i < 16 * kUnits; i += 64)
        *reinterpret_cast<uint4 *>(v + 8 * i) = make_uint4(0, 0, 0, 0);
    }
    // Keys with an infinity or NaN among their values that some rows of the block see
    // and others do not: 0 * NaN again. Their values are zeroed too, and added at the
    // end to the rows that see them.
    if (!prefix && tile.first_position != tile.last_position &&
        k0 + kKeys - 1 > tile.first_position) {
      uint16_t *v = tile_lds + stage * 2 * kPlane + kPlane + 16 * wave * kD;
      uint32_t odd_rows = 0;
#pragma unroll
      for (int i = 0; i < kOps; ++i) {
        const uint4 x = *reinterpret_cast<const uint4 *>(v + 8 * (64 * i + lane));
        const uint64_t odd = __ballot(nonfinite<T>(x.x) || nonfinite<T>(x.y) ||
                                      nonfinite<T>(x.z) || nonfinite<T>(x.w));
        if (odd != 0) {
#pragma unroll
          for (int r = 0; r < kOpRows; ++r)
            if ((odd >> (r * kUnits) & ((uint64_t{1} << kUnits) - 1)) != 0)
              odd_rows |= 1U << (kOpRows * i + r);
          if ((odd_rows >> (kOpRows * i + lane / kUnits) & 1) != 0)
            *reinterpret_cast<uint4 *>(v + 8 * (64 * i + lane)) = make_uint4(0, 0, 0, 0);
        }
      }
      if (odd_tiles == 0)
        odd_first = k0;
      if (lane == 0)
        odd_s[4 * odd_tiles + wave] = static_cast<uint16_t>(odd_rows);
      ++odd_tiles;
    }
    __syncthreads();
    if (k0 + kKeys < key1) {
      pages = pages_of(entries, k0 + kKeys);
      issue(k0 + kKeys, stage ^ 1, pages);
      entries = entries_at(k0 + 2 * kKeys);
    }
    if (!wave_rows || k0 > wave_last)
      continue;
    const uint16_t *k_s = tile_lds + stage * 2 * kPlane, *v_s = k_s + kPlane;

    // Operands are requested from LDS a part (a quarter of the tile's products) ahead of
    // their products: left to the compiler, the wave waits for each.
    constexpr int kPart = kSteps / 2;
    vec k_part[2][kPart], v_part[2][kTiles];
    const auto read_keys = [&](int kk) {
      const int r = 32 * (kk / 2) + col;
#pragma unroll
      for (int s = 0; s < kPart; ++s)
        k_part[kk % 2][s] = *reinterpret_cast<const vec *>(
            k_s + r * kD + 8 * swizzle_k<kUnits>(r, 2 * (kPart * (kk % 2) + s) + half));
    };
    f32x16 score[2];
    read_keys(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk < 3)
        read_keys(kk + 1);
      else
        read_values<T, kD>(v_s, 0, v_part[0]);
      __builtin_amdgcn_sched_barrier(0);
      if (kk % 2 == 0)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          score[kk / 2][e] = 0.0F;
#pragma unroll
      for (int s = 0; s < kPart; ++s)
        score[kk / 2] = Mfma<T>::run(k_part[kk % 2][s], q[kPart * (kk % 2) + s], score[kk / 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (missing != 0 || k0 + kKeys - 1 > wave_first || k0 + kKeys > key1) {
      const int visible = min(position + 1, key1) - k0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = 32 * u + (e >> 2) * 8 + 4 * half + (e & 3);
          score[u][e] = key < visible && (missing >> (2 * u + e / 8) & 1) == 0 ? score[u][e]
                                                                               : -INFINITY;
        }
    }
    float tile_top = score[0][0];
#pragma unroll
    for (int e = 1; e < 16; ++e)
      tile_top = fmaxf(tile_top, score[0][e]);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      tile_top = fmaxf(tile_top, score[1][e]);
    tile_top = fmaxf(tile_top, __shfl_xor(tile_top, 32, 64));
    const bool follows = (tile_top - top) * a.scale2 > kSlack<T>;
    if (__any(follows)) {
      const float next = follows ? tile_top : top;
      const float shrink = follows ? weight(top, next, a.scale2) : 1.0F;
      sum *= shrink;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          out[t][e] *= shrink;
      top = next;
      const bool far = is_far(top, a.scale2);
      far_rows = __any(far);
      shift = far || top == -INFINITY ? kLift<T> : fmaf(-top, a.scale2, kLift<T>);
    }
    if (far_rows) {
      const float base = is_far(top, a.scale2) ? top : 0.0F;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          score[u][e] -= base;
    }
    vec p[2];
    const auto weights = [&](int kk) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        p[kk % 2][j] = static_cast<T>(
            __builtin_amdgcn_exp2f(fmaf(score[kk / 2][8 * (kk % 2) + j], a.scale2, shift)));
      sum = Mfma<T>::add(p[kk % 2], sum);
    };
    weights(0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk < 3)
        read_values<T, kD>(v_s, kk + 1, v_part[(kk + 1) % 2]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        out[t] = Mfma<T>::run(v_part[kk % 2][t], p[kk % 2], out[t]);
      if (kk < 3)
        weights(kk + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The odd keys' values, to the rows that see them (their weights are in the sum).
  if (odd_tiles > 0) {
    __syncthreads();
    for (int i = 0; i < 4 * odd_tiles; ++i)
      for (uint32_t bits = odd_s[i]; bits != 0; bits &= bits - 1) {
        const int key = odd_first + 16 * i + __builtin_ctz(bits);
        const int page = checked_page(table, key >> a.cache.page_shift, a.cache.pages);
        if (page < 0)
          continue;
        const size_t at = page * a.cache.page_stride + work.kv_head * a.cache.head_stride +
                          (key & slot_mask) * a.cache.token_stride;
        const uint16_t *k = a.cache.keys + at + 8 * half, *v = a.cache.values + at + 4 * half;
        // The score as it was: the same instructions, the key in all of their 32 rows. (A
        // sum in another order is another one, by any factor in the weight of a far score.)
        f32x16 score;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          score[e] = 0.0F;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          score = Mfma<T>::run(*reinterpret_cast<const vec *>(k + 16 * s), q[s], score);
        const float w = lifted<T>(score[0], top, a.scale2);
        if (key <= position) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              out[t][e] = fmaf(w, element<T>(v[32 * t + (e >> 2) * 8 + (e & 3)]), out[t][e]);
        }
      }
  }

  const float total = sum + __shfl_xor(sum, 32, 64);
  if (!active)
    return;
  // Entry e of tile t: element 32t + 8 * (e / 4) + 4 half + e % 4 of row `row`.
  if (!prefix && single_chunk(a, position)) {
    if (work.chunk > 0)
      return;
    // A row without keys is zero.
    const float inverse = total > 0.0F ? 1.0F / total : total == 0.0F ? 0.0F : total;
    uint16_t *dst = a.out + token * a.out_stride + head * kD + 4 * half;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        uint16_t bits[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          bits[j] = bits_of<T>(out[t][e + j] * inverse);
        *reinterpret_cast<uint2 *>(dst + 32 * t + 2 * e) = __builtin_bit_cast(uint2, bits);
      }
    return;
  }
  if (key0 > position)
    return;  // no key of the chunk is the row's, and no one reads its slot
  const size_t slot =
      (token * a.heads + head) * a.slots + (prefix ? work.chunk : a.prefix_slots + work.chunk);
  if (half == 0)
    a.state[slot] = make_float2(top, total);
  float *dst = a.part + slot * kD + 4 * half;
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4 *>(dst + 32 * t + 2 * e) =
          make_float4(out[t][e], out[t][e + 1], out[t][e + 2], out[t][e + 3]);
}

// ------------------------------------------------------------- launches
// LDS of a 128-row block: two stages of K and V, and a word for each 16 keys of the
// tiles that only some of its rows see (four: 128 positions and a tile's rest).
constexpr size_t tile_lds_bytes(size_t head_dim) {
  return 2 * 2 * 64 * head_dim * sizeof(uint16_t) + 16 * sizeof(uint16_t);
}
static_assert(2 * tile_lds_bytes(128) <= 160 * 1024, "two blocks per CU");

// Blocks of a launch. kSmall: 16 rows; kLarge: 128 rows; kMixed: 128 rows on the shared
// keys beside 16 rows on each sequence's own.
enum BlockKind : int { kSmall, kLarge, kMixed };
template <typename T, int kD, int kKind>
__global__ __launch_bounds__(256, kKind == kSmall ? 3 : 2) void
paged_attention_kernel(const AttendArgs a, unsigned prefix_blocks) {
  extern __shared__ __attribute__((aligned(16))) uint16_t attend_lds[];
  if (blockIdx.x == prefix_blocks)
    report_bad_sequences(a.batch);
  const BlockWork work = block_work(a, prefix_blocks);
  if (kKind == kLarge || (kKind == kMixed && work.prefix))
    tile_block<T, kD>(a, work, attend_lds);
  else
    stream_block<T, kD>(a, work, *reinterpret_cast<StreamShared<kD> *>(attend_lds));
}

// Rows whose keys lay in several chunks: the chunks rescaled to their common
// maximum and summed in a fixed order. A wave's lanes hold four elements of a row
// each, its groups of kD / 4 lanes every kGroups-th chunk, and lane l the states of
// chunks l, 64 + l, .. (256 at most). kSplit: a block per row and head, its four
// waves sharing the chunks; else a block takes `heads` heads of one row, a wave
// every fourth of them, so that a batch of many rows looks a row up once. Its bytes
// bound it where rows are many (1989 tokens of 15 heads and two chunks 14 us), else the
// launch and the loads that wait for each other, 4 to 5 us.
template <typename T, int kD, bool kSplit>
__global__ __launch_bounds__(256) void paged_combine_kernel(const AttendArgs a, int heads) {
  constexpr int kLanes = kD / 4, kGroups = 64 / kLanes, kStates = kSplit ? 4 : 1;
  constexpr int kWaves = kSplit ? 4 : 1;  // of a row and head
  __shared__ float4 out_s[4][kLanes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head_blocks = (a.heads + heads - 1) / heads;
  const int token = static_cast<int>(blockIdx.x / head_blocks);
  const int head0 = static_cast<int>(blockIdx.x % head_blocks) * heads;
  const int sub = kSplit ? wave : 0, group = lane / kLanes, l = lane % kLanes;
  const int sequence = sequence_of(a.batch, token);
  if (sequence < 0)
    return;
  const SequenceRows rows = sequence_rows(a.batch, sequence);
  const int position = rows.length - rows.count + token - rows.first;
  if (!rows.valid || single_chunk(a, position))
    return;
  // (A row behind the prefix sees it all, a padding row nothing.)
  const int count = position < 0 ? 0 : a.prefix_slots + own_chunks(a, position);
  for (int head = head0 + (kSplit ? 0 : wave); head < min(a.heads, head0 + heads);
       head += kSplit ? 1 : 4) {
    const size_t at = static_cast<size_t>(token) * a.heads + head;
    const float *src = a.part + at * a.slots * kD + 4 * l;
    float top[kStates], total = 0.0F, all = -INFINITY;
    float part_sum[kStates];
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
      const bool has = 64 * i + lane < count;
      const float2 s = has ? a.state[at * a.slots + 64 * i + lane] : make_float2(-INFINITY, 0.0F);
      top[i] = s.x;
      part_sum[i] = s.y;
      all = fmaxf(all, top[i]);
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
      all = fmaxf(all, __shfl_xor(all, offset, 64));
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
      // (A chunk without visible keys has no weight.)
      top[i] = top[i] == -INFINITY ? 0.0F : weight(top[i], all, a.scale2);
      total = fmaf(part_sum[i], top[i], total);
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
      total += __shfl_xor(total, offset, 64);
    float4 o = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
      const int end = min(64, count - 64 * i);
      for (int c0 = kGroups * sub; c0 < end; c0 += 4 * kGroups * kWaves) {
        float scale[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + kGroups * kWaves * u + group;
          scale[u] = __shfl(top[i], c & 63, 64);
          v[u] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
          if (c < end)
            v[u] = *reinterpret_cast<const float4 *>(src + (64 * i + c) * kD);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          o.x = fmaf(v[u].x, scale[u], o.x);
          o.y = fmaf(v[u].y, scale[u], o.y);
          o.z = fmaf(v[u].z, scale[u], o.z);
          o.w = fmaf(v[u].w, scale[u], o.w);
        }
      }
    }
#pragma unroll
    for (int offset = kLanes; offset < 64; offset <<= 1) {
      o.x += __shfl_xor(o.x, offset, 64);
      o.y += __shfl_xor(o.y, offset, 64);
      o.z += __shfl_xor(o.z, offset, 64);
      o.w += __shfl_xor(o.w, offset, 64);
    }
    if constexpr (kSplit) {
      if (lane < kLanes)
        out_s[wave][l] = o;
      __syncthreads();
      if (wave != 0)
        return;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        const float4 v = out_s[w][l];
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
      }
    }
    const float inverse = total > 0.0F ? 1.0F / total : total == 0.0F ? 0.0F : total;
    const uint16_t bits[4] = {bits_of<T>(o.x * inverse), bits_of<T>(o.y * inverse),
                              bits_of<T>(o.z * inverse), bits_of<T>(o.w * inverse)};
    if (lane < kLanes)
      *reinterpret_cast<uint2 *>(a.out + token * a.out_stride + head * kD + 4 * l) =
          __builtin_bit_cast(uint2, bits);
  }
}

struct AttendPlan {
  bool own_stream, prefix_stream;  // 16-row blocks, else 128-row ones
  size_t tiles, prefix_tiles;      // row tiles of the own keys, of the shared ones
  int chunk, prefix_chunk, prefix_slots, slots;
};
constexpr size_t kMostSlots = 128;  // of each phase (256 in the combining kernel)

// Chunks of a row of least .. most keys, every number as likely, on average: the sum
// over k of the chance that it has more than k * chunk.
double mean_chunks(double least, double most, double chunk) {
  const double all = std::ceil(least / chunk), any = std::ceil(most / chunk);
  return any <= all ? all
                    : all + (any - all) * (most - 0.5 * (all + any - 1.0) * chunk) / (most - least);
}

// What the parts of one phase may take, in bytes: half of the last cache. One chunk
// is always taken.
constexpr double kMostPartBytes = 128e6;

// The 16-row blocks of a phase: `blocks` of them for each chunk of the longest row's
// `most` keys; the rows see as many each, or, uneven, anything up to that.
struct StreamPhase {
  size_t most, blocks;
  bool uneven;
  bool joined;  // parts are joined in any case
  double all_part_bytes;
};

// Keys per block of the 16-row kernel: the split of least modelled time, its constants
// fitted to measured splits (3% on average behind the best split of each of 49 batches,
// 26% at most: 4 sequences of up to 6000 keys, 21.6 us for 17.1). Keys and values stream at 5.8 TB/s from 160 blocks on; 1000 keys take
// a block 10 us, and 8 at the end, while the chip runs empty; a part's block costs
// 3 ns and joining the parts 9 us. Chunks are 128 keys and more, 32 for each wave.
int stream_chunk(const StreamPhase &phase, size_t head_dim) {
  const double most = static_cast<double>(phase.most), least = phase.uneven ? 0.0 : most;
  const double bytes = 2.0 * (least + most) * static_cast<double>(phase.blocks * head_dim);
  int best = 0;
  double best_us = 0.0;
  for (size_t slots = 1; slots <= kMostSlots; slots += slots / 16 + 1) {
    const int chunk = static_cast<int>((phase.most + slots * 128 - 1) / (slots * 128) * 128);
    if (best != 0 && static_cast<double>(slots) * phase.all_part_bytes > kMostPartBytes)
      break;
    const double blocks = mean_chunks(least, most, chunk) * static_cast<double>(phase.blocks);
    const double full = static_cast<double>(std::min<size_t>(chunk, phase.most));
    double us = std::max(bytes / (5.8e6 * std::min(1.0, blocks / 160.0)), 0.010 * full) +
                0.008 * full * std::min(1.0, blocks / 444.0);
    if (static_cast<size_t>(chunk) < phase.most)
      us += (phase.joined ? 0.0 : 9.0) + 0.003 * blocks;
    if (best == 0 || us < best_us) {
      best = chunk;
      best_us = us;
    }
    if (chunk == 128)
      break;
  }
  return best;
}

// The 128-row blocks of a phase: `tiles` of them see `least` .. `most` keys each,
// evenly spread, and all together read kv_bytes of keys and values and leave a part
// of part_bytes in each chunk; all rows of the batch have all_part_bytes each.
struct TilePhase {
  size_t tiles, least, most;
  double other_keys;  // keys of further blocks, all together
  double kv_bytes, part_bytes, all_part_bytes;
};

// Keys per block: the split of least modelled time, its constants fitted to measured
// splits (4% on average behind the best split of each of 40 batches, 28% at most: 16
// ragged sequences of up to 64 tokens on 2000, 46 us for 36). 64 keys of head_dim 128
// take a block 2.3 us where two share a CU and 2.1 alone (in the middle of a long
// chunk the kernel now measures 2.1 and 1.2: of a lone block the model is least true);
// 512 blocks run at a time, the longest start first, and the last ones leave part of
// the chip idle. Keys and values stream at 5 TB/s from 512 blocks, at 3.6 from one
// a CU. A part costs its bytes at 1.3 TB/s (written, read again, more tails), and all
// parts one more launch.
int tile_chunk(const TilePhase &phase, size_t head_dim) {
  const double key_us = 2.3 / 64.0 * static_cast<double>(head_dim) / 128.0;
  constexpr double kAlone = 0.9;
  int best = 0;
  double best_us = 0.0;
  for (size_t half_chunks = 2; half_chunks <= 2 * kMostSlots; half_chunks += half_chunks / 16 + 1) {
    // chunks of the longest rows: 1, 1.5, 2, ..
    const size_t longest_keys = (2 * phase.most + half_chunks - 1) / half_chunks;
    const int chunk = static_cast<int>((longest_keys + 63) / 64 * 64);
    const size_t slots = (phase.most + chunk - 1) / chunk;
    if (best != 0 && (chunk < 128 || slots > kMostSlots ||
                      static_cast<double>(slots) * phase.all_part_bytes > kMostPartBytes))
      break;
    const double chunks = mean_chunks(static_cast<double>(phase.least),
                                      static_cast<double>(phase.most), chunk);
    const double keys = 0.5 * static_cast<double>((phase.least + phase.most) * phase.tiles) +
                        phase.other_keys;
    const double full = static_cast<double>(std::min<size_t>(chunk, phase.most));
    const double least = static_cast<double>(std::min<size_t>(chunk, phase.least));
    const double own_blocks = chunks * static_cast<double>(phase.tiles);
    const double rounds = (own_blocks + phase.other_keys / full) / 512.0;
    const double pairs = std::clamp(2.0 * rounds - 1.0, 0.0, 1.0);  // CUs with two blocks
    double us = full * key_us * (kAlone + (1.0 - kAlone) * pairs);
    if (rounds > 0.5)
      us = std::max(us, (keys / 512.0 + (std::ceil(rounds) - rounds) * least) * key_us);
    us = std::max(us, phase.kv_bytes /
                          (3.6e6 + 1.4e6 * std::clamp(own_blocks / 256.0 - 1.0, 0.0, 1.0)));
    if (chunks > 1.0)
      us += 5.0 + phase.part_bytes * chunks / 1.3e6;
    if (best == 0 || us < best_us) {
      best = chunk;
      best_us = us;
    }
  }
  return best;
}

AttendPlan plan_attention(const PagedCache &cache, const PagedBatch &batch, size_t heads) {
  const size_t kv = static_cast<size_t>(cache.kv_heads), group = heads / kv;
  const size_t sequences = static_cast<size_t>(batch.sequences);
  const size_t tokens = static_cast<size_t>(batch.tokens);
  const size_t dim = static_cast<size_t>(cache.head_dim);
  const size_t most = static_cast<size_t>(batch.max_tokens) * group;
  AttendPlan plan{};
  plan.own_stream = most <= 16;
  plan.prefix_stream = tokens * group <= 16;
  const size_t rows = plan.own_stream ? 16 : 128;
  // A tile each for the rows that fill one, and one more for each sequence's rest.
  plan.tiles = plan.own_stream ? sequences
                               : std::min(sequences * ((most + rows - 1) / rows),
                                          tokens * group / rows + std::min(sequences, tokens));
  const size_t own = std::max(1, batch.max_length - batch.shared_length);
  const double part_bytes = static_cast<double>(tokens * heads * dim * sizeof(float));
  if (plan.own_stream) {
    plan.chunk = stream_chunk(
        {own, plan.tiles * kv, sequences > 1, batch.shared_length > 0, part_bytes}, dim);
  } else {
    // The longest sequence is taken to bring the most rows too; the others' lengths
    // are not known here and count as 0.6 of its.
    const size_t longest_tiles = (most + rows - 1) / rows;
    const double share = static_cast<double>(batch.max_tokens) / static_cast<double>(tokens);
    plan.chunk = tile_chunk({longest_tiles * kv, own - std::min(own, most / group) + 1, own,
                             0.6 * static_cast<double>((plan.tiles - longest_tiles) * kv) *
                                 static_cast<double>(own),
                             4.0 * static_cast<double>(own * kv * dim), part_bytes * share,
                             part_bytes},
                            dim);
  }
  const int own_slots = static_cast<int>((own + plan.chunk - 1) / plan.chunk);
  if (batch.shared_length > 0) {
    const size_t shared = static_cast<size_t>(batch.shared_length);
    const size_t prefix_rows = plan.prefix_stream ? 16 : 128;
    plan.prefix_tiles = (tokens * group + prefix_rows - 1) / prefix_rows;
    plan.prefix_chunk =
        plan.prefix_stream
            ? stream_chunk({shared, plan.prefix_tiles * kv, false, true, part_bytes}, dim)
            : tile_chunk({plan.prefix_tiles * kv, shared, shared, 0.0,
                          4.0 * static_cast<double>(shared * kv * dim), part_bytes, part_bytes},
                         dim);
    plan.prefix_slots =
        static_cast<int>((shared + plan.prefix_chunk - 1) / plan.prefix_chunk);
  }
  plan.slots = plan.prefix_slots + own_slots;
  return plan;
}

size_t plan_bytes(const AttendPlan &plan, const PagedCache &cache, const PagedBatch &batch,
                  size_t heads) {
  return plan.slots == 1 ? 0
                         : static_cast<size_t>(batch.tokens) * heads * plan.slots *
                               (cache.head_dim + 2) * sizeof(float);
}

template <typename T, int kD>
Status launch_attention(const AttendArgs &args, const AttendPlan &plan, hipStream_t stream) {
  const size_t kv = static_cast<size_t>(args.cache.kv_heads);
  const size_t prefix_blocks = plan.prefix_tiles * kv * plan.prefix_slots;
  const size_t blocks = prefix_blocks + plan.tiles * kv * (plan.slots - plan.prefix_slots);
  // A launch counts its threads in 32 bits.
  const size_t tokens = static_cast<size_t>(args.batch.tokens), heads = args.heads;
  // A block per row and head where there are more chunks than lanes, or many chunks of
  // few rows: 512 rows of 31 chunks 4.0 us, else 6.4; 600 tokens' rows of few chunks 103
  // us with the attention, else 81.
  const bool split_join = plan.slots > 64 || (plan.slots > 16 && tokens * heads <= 2048);
  // Four heads of a row per joining block, all of them where the rows fill the chip.
  const size_t of_block =
      split_join ? 1 : std::min(heads, 4 * std::max<size_t>(1, tokens * heads / 8192));
  const size_t join_blocks = plan.slots == 1 ? 0 : tokens * ceil_div(heads, of_block);
  constexpr size_t kMostThreads = (size_t{1} << 32) - 1;
  if (blocks > kMostThreads / 256 || join_blocks > kMostThreads / 256)
    return {ErrorCode::kInvalidArgument, "paged_attention: grid too large"};
  auto kernel = paged_attention_kernel<T, kD, kLarge>;
  size_t lds = tile_lds_bytes(kD);
  if (plan.own_stream && (plan.prefix_stream || prefix_blocks == 0)) {
    kernel = paged_attention_kernel<T, kD, kSmall>;
    lds = sizeof(StreamShared<kD>);
  } else if (plan.own_stream) {
    kernel = paged_attention_kernel<T, kD, kMixed>;
    lds = std::max(lds, sizeof(StreamShared<kD>));
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds,
                     stream, args, static_cast<unsigned>(prefix_blocks));
  EVO_TRY(launch_status("paged_attention_kernel"));
  if (plan.slots == 1)
    return Status::Ok();
  const auto join = split_join ? paged_combine_kernel<T, kD, true>
                               : paged_combine_kernel<T, kD, false>;
  hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(join_blocks)), dim3(256), 0, stream, args,
                     static_cast<int>(of_block));
  return launch_status("paged_combine_kernel");
}

template <typename T>
Status launch_dim(const AttendArgs &args, const AttendPlan &plan, hipStream_t stream) {
  switch (args.cache.head_dim) {
  case 32: return launch_attention<T, 32>(args, plan, stream);
  case 64: return launch_attention<T, 64>(args, plan, stream);
  default: return launch_attention<T, 128>(args, plan, stream);
  }
}

}  // namespace

size_t paged_attention_workspace_bytes(const PagedCache &cache, const PagedBatch &batch,
                                       size_t heads) {
  const size_t kv = static_cast<size_t>(cache.kv_heads);
  if (heads == 0 || heads % kv != 0 || heads > (1U << 16))
    return 0;
  return plan_bytes(plan_attention(cache, batch, heads), cache, batch, heads);
}

Status paged_attention(const PagedCache &cache, const PagedBatch &batch, const void *query,
                       size_t query_stride, size_t heads, float scale, void *out,
                       size_t out_stride, void *workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  const size_t kv = static_cast<size_t>(cache.kv_heads), dim = static_cast<size_t>(cache.head_dim);
  if (query == nullptr || out == nullptr || heads == 0 || heads > (1U << 16) || heads % kv != 0)
    return {ErrorCode::kInvalidArgument,
            "paged_attention: null tensor, or heads that are no multiple of kv_heads"};
  if ((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
      (query_stride | out_stride) % 8 != 0 || query_stride < heads * dim ||
      out_stride < heads * dim)
    return {ErrorCode::kInvalidArgument,
            "paged_attention: rows have to start on 16 bytes and hold every head"};
  if (out == query && out_stride != query_stride)
    return {ErrorCode::kInvalidArgument,
            "paged_attention: in place, out_stride has to be query_stride"};
  const float scale2 = 1.4426950408889634F * scale;
  if (!(scale > 0.0F) || !std::isfinite(scale2))
    return {ErrorCode::kInvalidArgument, "paged_attention: scale must be positive, and its multiple by log2(e) finite"};
  // (Rows are counted in 32 bits, up to the end of their last tile.)
  if (static_cast<size_t>(batch.tokens) * heads >= (size_t{1} << 31) - 128)
    return {ErrorCode::kInvalidArgument, "paged_attention: too many rows"};
  const AttendPlan plan = plan_attention(cache, batch, heads);
  const size_t bytes = plan_bytes(plan, cache, batch, heads);
  if (bytes != 0 && (workspace == nullptr || workspace_bytes < bytes ||
                     reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return {ErrorCode::kInvalidArgument,
            "paged_attention: workspace too small (" + std::to_string(bytes) +
                " bytes needed) or not 16-byte aligned"};
  const AttendArgs args{cache, batch, static_cast<const uint16_t *>(query), query_stride,
                        static_cast<uint16_t *>(out), out_stride, static_cast<int>(heads),
                        static_cast<int>(heads / kv), scale2, plan.chunk,
                        plan.prefix_chunk, plan.prefix_slots, plan.slots,
                        plan.own_stream ? 1 : 0,
                        static_cast<float *>(workspace),
                        reinterpret_cast<float2 *>(static_cast<float *>(workspace) +
                                                   static_cast<size_t>(batch.tokens) * heads *
                                                       plan.slots * dim)};
  return cache.dtype == kElementBF16 ? launch_dim<__bf16>(args, plan, stream)
                                     : launch_dim<_Float16>(args, plan, stream);
}

}  // namespace evo::hip
