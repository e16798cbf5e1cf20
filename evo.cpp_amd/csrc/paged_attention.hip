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
// Scores, maxima, sums and outputs are F32; the weights p <= 1 are rounded to the
// cache's type for the second product, and the sum is taken of the rounded ones,
// so that the weights applied add up to one.
#include "common.hpp"
#include "ops.hpp"
#include "paged.hpp"

#include <algorithm>
#include <cmath>

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
  int chunk;          // own keys per chunk (a multiple of 128)
  int prefix_chunk;   // shared keys per chunk
  int prefix_slots;   // chunks of the shared keys
  int slots;          // chunks of a row at most, the shared ones first
  float *part;        // [tokens][heads][slots][2 + head_dim]
};

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  typedef bf16x8 vec;
  static __device__ inline f32x4 run(const vec &a, const vec &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<_Float16> {
  typedef f16x8 vec;
  static __device__ inline f32x4 run(const vec &a, const vec &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <typename T> __device__ inline uint16_t bits_of(float v) {
  return __builtin_bit_cast(uint16_t, static_cast<T>(v));
}

// Chunks of a row at `position` (-1 and below: it sees nothing).
__device__ inline int own_chunks(const AttendArgs &a, int position) {
  const int keys = position + 1 - a.batch.shared_length;
  return keys <= 0 ? 0 : (keys + a.chunk - 1) / a.chunk;
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
      const int at = __builtin_ctzll(found);
      *sequence = s0 + at;
      *tile_in = tile - base - __shfl(through - tiles, at, 64);
      return true;
    }
    base += __shfl(through, 63, 64);
  }
  return false;
}

// Softmax state and output of 16 rows over the keys a wave has seen. Lane l:
// row l % 16, output elements kVec * (4 * (l / 16) + i) + t for i < 4, t < kVec.
template <int kD> struct RowState {
  static constexpr int kVec = kD / 16;
  float top, sum;  // log2 domain; the sum of this lane's own keys
  f32x4 out[kVec];
};

// One 32-key step. k[u][s]: K operand of keys 16u .., elements 32s ..; v[j]: this
// lane's 8 keys, kVec elements each.
template <typename T, int kD> struct Step {
  static constexpr int kVec = kD / 16, kSteps = kD / 32;
  typedef typename Mfma<T>::vec vec;
  vec k[2][kSteps];
  uint32_t v[8][kVec / 2];
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

// Loads the keys k0 .. k0 + 31 (pages page[0], page[1] of 16 each; -1: none, the
// registers are zeroed). k0 is a multiple of 16, so 16 keys share a page.
template <typename T, int kD>
__device__ inline void load_step(const AttendArgs &a, int kv_head, int k0, const int (&page)[2],
                                 Step<T, kD> &step) {
  using S = Step<T, kD>;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int mask = (1 << a.cache.page_shift) - 1;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (page[u] < 0) {
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s)
        step.k[u][s] = typename S::vec{};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < S::kVec / 2; ++w)
          step.v[4 * u + i][w] = 0;
      continue;
    }
    const size_t base = page[u] * a.cache.page_stride + kv_head * a.cache.head_stride +
                        ((k0 + 16 * u) & mask) * a.cache.token_stride;
    const uint16_t *k = a.cache.keys + base + col * a.cache.token_stride + 8 * g;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
      step.k[u][s] = *reinterpret_cast<const typename S::vec *>(k + 32 * s);
    const uint16_t *v = a.cache.values + base + 4 * g * a.cache.token_stride + S::kVec * col;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_words(v + i * a.cache.token_stride, step.v[4 * u + i]);
  }
}

// Adds a step's keys to 16 rows. visible: keys of the step this lane's row sees
// (of each 16: its number may be over 16 or below 0); limit: keys of the step that
// any row sees, whose values alone may be read.
template <typename T, int kD>
__device__ inline void attend(const Step<T, kD> &step, const typename Mfma<T>::vec *q,
                              float scale2, bool masked, const int (&visible)[2],
                              RowState<kD> &state) {
  using S = Step<T, kD>;
  const int g = (threadIdx.x & 63) >> 4;
  f32x4 score[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    score[u] = f32x4{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
      score[u] = Mfma<T>::run(step.k[u][s], q[s], score[u]);
  }
  if (masked) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        score[u][i] = 4 * g + i < visible[u] ? score[u][i] : -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = fmaxf(top, score[u][i]);
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64)) * scale2;
  const float next = fmaxf(state.top, top);
  if (__any(next != state.top)) {
    const float shrink = next == -INFINITY ? 1.0F : __builtin_amdgcn_exp2f(state.top - next);
    state.sum *= shrink;
#pragma unroll
    for (int t = 0; t < S::kVec; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        state.out[t][i] *= shrink;
    state.top = next;
  }
  const float base = next == -INFINITY ? 0.0F : next;
  typename S::vec p;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T w = static_cast<T>(__builtin_amdgcn_exp2f(fmaf(score[u][i], scale2, -base)));
      p[4 * u + i] = w;
      state.sum += static_cast<float>(w);
    }
#pragma unroll
  for (int t = 0; t < S::kVec; ++t) {
    // Element t of this lane's kVec of each of its 8 keys.
    uint32_t word[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      word[j] = __builtin_amdgcn_perm(step.v[2 * j + 1][t / 2], step.v[2 * j][t / 2],
                                      t % 2 == 0 ? 0x05040100U : 0x07060302U);
    state.out[t] = Mfma<T>::run(__builtin_bit_cast(typename S::vec, word), p, state.out[t]);
  }
}

// 16 rows of a key/value head and a chunk of their keys per block; its four
// waves take every fourth 32-key step and join their states through LDS.
// Blocks below prefix_blocks take the shared keys, rows of the whole batch.
template <typename T, int kD>
__global__ __launch_bounds__(256) void paged_stream_kernel(const AttendArgs a,
                                                           unsigned prefix_blocks) {
  constexpr int kRows = 16, kWaves = 4, kVec = kD / 16, kSteps = kD / 32;
  typedef typename Mfma<T>::vec vec;
  __shared__ float top_s[kWaves][kRows], sum_s[kWaves][kRows];
  __shared__ __attribute__((aligned(16))) float out_s[kWaves][kRows][kD + 4];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool prefix = blockIdx.x < prefix_blocks;
  const int kv = a.cache.kv_heads;
  unsigned rest = prefix ? blockIdx.x : blockIdx.x - prefix_blocks;
  const int kv_head = static_cast<int>(rest % kv);
  rest /= kv;
  const int chunks = prefix ? a.prefix_slots : a.slots - a.prefix_slots;
  const int chunk = static_cast<int>(rest % chunks);
  const int tile = static_cast<int>(rest / chunks);

  if (blockIdx.x == prefix_blocks)
    report_bad_sequences(a.batch);

  // Rows of the tile: `row` of `rows` at this lane, token and query head.
  int row0, rows, first_token, first_position, last_position, sequence = 0;
  if (prefix) {
    row0 = tile * kRows;
    rows = a.batch.tokens * a.group;
    first_token = 0;
    first_position = last_position = a.batch.shared_length - 1;
  } else {
    int tile_in;
    if (!find_tile<kRows>(a, tile, &sequence, &tile_in))
      return;
    sequence = __builtin_amdgcn_readfirstlane(sequence);
    const SequenceRows own = sequence_rows(a.batch, sequence);
    row0 = __builtin_amdgcn_readfirstlane(tile_in) * kRows;
    rows = own.count * a.group;
    first_token = own.first;
    first_position = own.length - own.count + row0 / a.group;
    last_position = own.length - own.count + (min(row0 + kRows, rows) - 1) / a.group;
  }
  const int row = row0 + col;
  const bool active = row < rows;
  const int token_in = (active ? row : row0) / a.group;
  const int token = first_token + token_in;
  const int head = kv_head * a.group + (active ? row : row0) % a.group;
  const int position = prefix ? last_position : first_position + token_in - row0 / a.group;

  const int key0 = prefix ? chunk * a.prefix_chunk : a.batch.shared_length + chunk * a.chunk;
  const int key1 = min(last_position + 1, key0 + (prefix ? a.prefix_chunk : a.chunk));
  if (key0 >= key1 && (prefix || chunk > 0 || a.slots > 1))
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
                                : a.batch.page_table + sequence * a.batch.table_stride;
  for (int k0 = key0 + 32 * wave; k0 < key1; k0 += 32 * kWaves) {
    int page[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      page[u] = -1;
      if (k0 + 16 * u < key1) {
        page[u] = checked_page(table, (k0 + 16 * u) >> a.cache.page_shift, a.cache.pages);
        if (page[u] < 0 && lane == 0)
          report(a.batch, kBadPage);
      }
      page[u] = __builtin_amdgcn_readfirstlane(page[u]);
    }
    Step<T, kD> step;
    load_step<T, kD>(a, kv_head, k0, page, step);
    const bool masked = page[0] < 0 || page[1] < 0 || k0 + 31 > first_position || k0 + 32 > key1;
    int visible[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int from = k0 + 16 * u;
      visible[u] = page[u] < 0 ? 0 : min(position + 1, key1) - from;
      // Values no row of the tile sees may be anything, and 0 * NaN is NaN.
      if (masked && from + 16 > key1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (from + 4 * g + i >= key1) {
#pragma unroll
            for (int w = 0; w < kVec / 2; ++w)
              step.v[4 * u + i][w] = 0;
          }
      }
    }
    attend<T, kD>(step, q, a.scale2, masked, visible, state);
  }

  // Join the four waves: each leaves its rows' maximum, sum and output.
  float sum = state.sum + __shfl_xor(state.sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (g == 0) {
    top_s[wave][col] = state.top;
    sum_s[wave][col] = sum;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < kVec; ++t)
      out_s[wave][col][kVec * (4 * g + i) + t] = state.out[t][i];
  __syncthreads();
  // Thread: row tid / 16, elements kVec * (tid % 16) ...
  const int r = threadIdx.x >> 4, d = kVec * (threadIdx.x & 15);
  if (row0 + r >= rows)
    return;
  float top = top_s[0][r];
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
    top = fmaxf(top, top_s[w][r]);
  float total = 0.0F, o[kVec] = {};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float scale = top_s[w][r] == -INFINITY ? 0.0F
                                                 : __builtin_amdgcn_exp2f(top_s[w][r] - top);
    total = fmaf(sum_s[w][r], scale, total);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      o[e] = fmaf(out_s[w][r][d + e], scale, o[e]);
  }
  const size_t out_token = first_token + (row0 + r) / a.group;
  const int out_head = kv_head * a.group + (row0 + r) % a.group;
  if (a.slots == 1) {
    // The row's only chunk. A row without keys is zero.
    const float inverse = total > 0.0F ? 1.0F / total : total == 0.0F ? 0.0F : total;
    uint16_t *dst = a.out + out_token * a.out_stride + out_head * kD + d;
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      dst[e] = bits_of<T>(o[e] * inverse);
    return;
  }
  const int slot = prefix ? chunk : a.prefix_slots + chunk;
  float *dst = a.part + ((out_token * a.heads + out_head) * a.slots + slot) * (kD + 2);
  if (d == 0) {
    dst[0] = top;
    dst[1] = total;
  }
#pragma unroll
  for (int e = 0; e < kVec; e += 2)
    *reinterpret_cast<float2 *>(dst + 2 + d + e) = make_float2(o[e], o[e + 1]);
}

// Rows whose keys lay in several chunks: a wave per row and head rescales the
// chunks to their common maximum and sums them in order, two elements a lane.
template <typename T, int kD>
__global__ __launch_bounds__(256) void paged_combine_kernel(const AttendArgs a) {
  const size_t index = blockIdx.x * 4ULL + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (index >= static_cast<size_t>(a.batch.tokens) * a.heads)
    return;
  const int token = static_cast<int>(index / a.heads), head = static_cast<int>(index % a.heads);
  const int sequence = sequence_of(a.batch, token);
  if (sequence < 0)
    return;
  const SequenceRows rows = sequence_rows(a.batch, sequence);
  if (!rows.valid || lane >= kD / 2)
    return;
  const int position = rows.length - rows.count + token - rows.first;
  const int own = own_chunks(a, position);
  // (Own keys and shared ones: a row behind the prefix has both, a padding row
  // neither.)
  const int count = position < 0 ? 0 : a.prefix_slots + own;
  const float *src = a.part + index * a.slots * (kD + 2);
  float top = -INFINITY;
  for (int c = 0; c < count; ++c)
    top = fmaxf(top, src[c * (kD + 2)]);
  float total = 0.0F, o0 = 0.0F, o1 = 0.0F;
#pragma unroll 4
  for (int c = 0; c < count; ++c) {
    const float *from = src + c * (kD + 2);
    const float scale = from[0] == -INFINITY ? 0.0F : __builtin_amdgcn_exp2f(from[0] - top);
    const float2 o = *reinterpret_cast<const float2 *>(from + 2 + 2 * lane);
    total = fmaf(from[1], scale, total);
    o0 = fmaf(o.x, scale, o0);
    o1 = fmaf(o.y, scale, o1);
  }
  const float inverse = total > 0.0F ? 1.0F / total : total == 0.0F ? 0.0F : total;
  uint16_t *dst = a.out + token * a.out_stride + head * kD + 2 * lane;
  dst[0] = bits_of<T>(o0 * inverse);
  dst[1] = bits_of<T>(o1 * inverse);
}

struct AttendPlan {
  size_t tiles, prefix_tiles;  // row tiles of the own keys, of the shared ones
  int chunk, prefix_chunk, prefix_slots, slots;
};

// Chunks of a launch: enough blocks for a few per CU, chunks of 128 keys and
// more (32 for each wave), at most 64 of a row.
int chunk_keys(size_t keys, size_t blocks) {
  const size_t wanted = std::max<size_t>(1, 2048 / std::max<size_t>(1, blocks));
  const size_t chunks = std::min<size_t>({wanted, (keys + 127) / 128, 64});
  return static_cast<int>((keys + chunks * 128 - 1) / (chunks * 128) * 128);
}

AttendPlan plan_attention(const PagedCache &cache, const PagedBatch &batch, size_t heads) {
  constexpr size_t kRows = 16;
  const size_t kv = static_cast<size_t>(cache.kv_heads), group = heads / kv;
  const size_t sequences = static_cast<size_t>(batch.sequences);
  const size_t tokens = static_cast<size_t>(batch.tokens);
  const size_t most = static_cast<size_t>(batch.max_tokens) * group;
  AttendPlan plan{};
  // A tile each for the rows that fill one, and one more for each sequence's rest.
  plan.tiles = std::min(sequences * ((most + kRows - 1) / kRows),
                        tokens * group / kRows + std::min(sequences, tokens));
  const size_t own = static_cast<size_t>(batch.max_length - batch.shared_length);
  plan.chunk = chunk_keys(std::max<size_t>(own, 1), plan.tiles * kv);
  int own_slots = static_cast<int>((std::max<size_t>(own, 1) + plan.chunk - 1) / plan.chunk);
  if (batch.shared_length > 0) {
    const size_t shared = static_cast<size_t>(batch.shared_length);
    plan.prefix_tiles = (tokens * group + kRows - 1) / kRows;
    plan.prefix_chunk = chunk_keys(shared, plan.prefix_tiles * kv);
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
  if (blocks >= (size_t{1} << 31))
    return {ErrorCode::kInvalidArgument, "paged_attention: grid too large"};
  hipLaunchKernelGGL((paged_stream_kernel<T, kD>), dim3(static_cast<unsigned>(blocks)), dim3(256),
                     0, stream, args, static_cast<unsigned>(prefix_blocks));
  EVO_TRY(launch_status("paged_stream_kernel"));
  if (plan.slots == 1)
    return Status::Ok();
  const size_t rows = static_cast<size_t>(args.batch.tokens) * args.heads;
  hipLaunchKernelGGL((paged_combine_kernel<T, kD>), dim3(ceil_div(rows, 4)), dim3(256), 0, stream,
                     args);
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
  if (!(scale > 0.0F) || !std::isfinite(scale))
    return {ErrorCode::kInvalidArgument, "paged_attention: scale must be positive and finite"};
  if (static_cast<size_t>(batch.tokens) * heads >= (size_t{1} << 31))
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
                        static_cast<int>(heads / kv), 1.4426950408889634F * scale, plan.chunk,
                        plan.prefix_chunk, plan.prefix_slots, plan.slots,
                        static_cast<float *>(workspace)};
  return cache.dtype == kElementBF16 ? launch_dim<__bf16>(args, plan, stream)
                                     : launch_dim<_Float16>(args, plan, stream);
}

}  // namespace evo::hip
