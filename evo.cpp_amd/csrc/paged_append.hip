// SPDX-License-Identifier: Apache-2.0
// Appends the keys and values of a batch's rows to the paged cache, rotated on
// the way, and writes the rotated queries.
//
// x' = x cos a - y sin a, y' = y cos a + x sin a over the rotated pairs of a
// query or key head, a = (position / scale) * inv_freq[i]; the rest and the
// values pass through. Bound by bytes: each value is read and written once. 8 prompts
// of up to 2048 tokens (F32 rows of 32 query, key and value heads of 128, 521 MB in
// all) take 101 us, 5.2 TB/s, the rate of a copy; one token takes 4.3 us, a launch and
// three loads that wait for each other (sequence, length, page).
//
// With norms, each query and key head x is first divided by its root mean square:
// x / (rms + eps) or x / sqrt(rms^2 + eps), times a scale of each element. The kDim / 16
// threads that hold a head add up its squares between themselves, in registers, which the
// loads hide: the same 8 prompts take 101 us, one token 4.6.
#include "common.hpp"
#include "ops.hpp"
#include "paged.hpp"

#include <cmath>

namespace evo::hip {

namespace {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

template <typename T> __device__ inline uint16_t to_bits(float v) {
  return __builtin_bit_cast(uint16_t, static_cast<T>(v));
}

template <typename S> __device__ inline float to_float(S v) { return static_cast<float>(v); }

// Eight consecutive elements: kVector where they start on 16 bytes.
template <typename S, bool kVector>
__device__ inline void load8(const S *src, float (&v)[8]) {
  if constexpr (!kVector) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = to_float(src[e]);
  } else if constexpr (sizeof(S) == 4) {
    const float4 a = *reinterpret_cast<const float4 *>(src);
    const float4 b = *reinterpret_cast<const float4 *>(src + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    typedef S S8 __attribute__((ext_vector_type(8)));
    const S8 a = *reinterpret_cast<const S8 *>(src);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = to_float(a[e]);
  }
}

template <typename T> __device__ inline void store8(uint16_t *dst, const float (&v)[8]) {
  u16x8 bits;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    bits[e] = to_bits<T>(v[e]);
  *reinterpret_cast<u16x8 *>(dst) = bits;
}

struct AppendArgs {
  PagedCache cache;
  PagedBatch batch;
  const void *projected;
  size_t row_stride;
  int heads;
  int column_split;
  const float *inv_freq;
  int rotary;       // elements of a head that turn
  int interleaved;
  float scale;
  uint16_t *query;
  size_t query_stride;
  int parts;        // blocks per row
};

// Cosine and sine of (position / scale) * inv_freq. The angle is formed and
// reduced to a turn in 64 bits: at position 10^6 a 32-bit product would be off
// by 0.06. The reduced turn holds its 24 bits in F32.
__device__ inline void turn(double position, float inv_freq, float *cosine, float *sine) {
  const double turns = position * static_cast<double>(inv_freq) * 0.15915494309189533577;
  sincospif(2.0F * static_cast<float>(turns - rint(turns)), sine, cosine);
}

// v of another lane of the wave, by the DPP control kCtrl: all lanes of a head run together.
template <int kCtrl> __device__ inline float other_lane(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_update_dpp(bits, bits, kCtrl, 0xf, 0xf, false));
}
// f over the 2, 4 or 8 neighbouring lanes that hold a head.
template <int kLanes, typename F> __device__ inline float over_head(float v, F f) {
  v = f(v, other_lane<0xb1>(v));  // quad_perm 1 0 3 2
  if constexpr (kLanes > 2)
    v = f(v, other_lane<0x4e>(v));  // quad_perm 2 3 0 1
  if constexpr (kLanes > 4)
    v = f(v, other_lane<0x141>(v));  // row_half_mirror: the other four of eight
  return v;
}

// What a head's elements are multiplied with to be normalized, but for their scale:
// first `lift` (a power of two, 1 but for squares that leave the range of F32), then
// `inverse`.
struct HeadSize {
  float lift, inverse;
};
template <int kLanes>
__device__ inline HeadSize head_size(const float (&u)[8], const float (&v)[8],
                                     const HeadNorm &norm) {
  constexpr float kMean = 1.0F / static_cast<float>(16 * kLanes);
  const auto squares = [&](float lift) {
    float sum = 0.0F;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = u[e] * lift, y = v[e] * lift;
      sum = fmaf(x, x, sum);
      sum = fmaf(y, y, sum);
    }
    return over_head<kLanes>(sum, [](float x, float y) { return x + y; });
  };
  const float sum = squares(1.0F);
  if (sum > 0x1p-100F && sum < 0x1p120F) {
    const float mean = sum * kMean;
    return {1.0F, 1.0F / (norm.inside ? sqrtf(mean + norm.eps) : sqrtf(mean) + norm.eps)};
  }
  // Squares beyond the range, infinities, NaN and zeros. The largest element is
  // brought near one; eps is at most 1, so it does not overflow. (Zeros are lifted too, as
  // 1 / eps may overflow where eps 2^120 is no small number.)
  float most = 0.0F;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    most = fmaxf(most, fmaxf(fabsf(u[e]), fabsf(v[e])));
  most = over_head<kLanes>(most, [](float x, float y) { return fmaxf(x, y); });
  const int power = most == 0.0F ? 120 : max(-126, min(-ilogbf(most), 120));
  const float lift = !(most < INFINITY) ? 1.0F : ldexpf(1.0F, power);
  const float rms = sqrtf(squares(lift) * kMean);
  const float size = norm.inside ? hypotf(rms, sqrtf(norm.eps) * lift) : rms + norm.eps * lift;
  return {lift, 1.0F / size};
}

// Which elements of a head a thread holds, in two groups of 8.
enum Layout : int {
  kHalves = 0,       // pairs (i, rotary / 2 + i), rotary % 16 == 0
  kInterleaved = 1,  // pairs (2i, 2i + 1)
  kAnyHalves = 2,    // pairs (i, rotary / 2 + i) of any even rotary
};

// A block takes one row, or with parts > 1 a part of its heads. kDim / 16
// threads hold a head's elements, 16 each, and keep their cosines over the
// heads that they walk. In halves thread j turns pairs 8j .. 8j + 7, groups at
// 8j and rotary / 2 + 8j, and threads past the rotated pairs hold what passes
// through; otherwise its groups lie side by side, and in halves of any size
// the partner of an element is loaded beside it.
template <typename S, typename T, int kDim, bool kVector, int kLayout, bool kNormed>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a,
                                                           const HeadNorm norm) {
  constexpr int kLanes = kDim / 16, kHeadsPerPass = 256 / kLanes;
  constexpr int kAngles = kLayout == kAnyHalves ? 16 : 8;
  const int row = static_cast<int>(blockIdx.x / a.parts);
  const int part = static_cast<int>(blockIdx.x % a.parts);
  if (blockIdx.x == 0)
    report_bad_sequences(a.batch);
  const int sequence = sequence_of(a.batch, row);
  if (sequence < 0)
    return;
  const SequenceRows rows = sequence_rows(a.batch, sequence);
  if (!rows.valid)
    return;
  const int position = rows.length - rows.count + (row - rows.first);
  int page = -1;
  if (position >= 0) {
    page = checked_page(a.batch.page_table + sequence * a.batch.table_stride,
                        position >> a.cache.page_shift, a.cache.pages);
    if (page < 0 && threadIdx.x == 0)
      report(a.batch, kBadPage);
  }
  const size_t at = page < 0 ? 0
                             : page * a.cache.page_stride +
                                   (position & ((1 << a.cache.page_shift) - 1)) *
                                       a.cache.token_stride;

  const int lane = threadIdx.x % kLanes;
  const int kv = a.cache.kv_heads, turned_heads = a.heads + kv, all_heads = turned_heads + kv;
  int head = threadIdx.x / kLanes + part * kHeadsPerPass;
  const int step = kHeadsPerPass * a.parts;
  const S *src = static_cast<const S *>(a.projected) + row * a.row_stride;
  const int half = a.rotary / 2;
  int first = 16 * lane, second = first + 8;
  bool turns = first < a.rotary;
  if (kLayout == kHalves) {
    turns = 8 * lane < half;
    if (turns) {
      first = 8 * lane;
      second = half + first;
    }
  }
  float cosine[kAngles], sine[kAngles];
  const double scaled = static_cast<double>(position) / static_cast<double>(a.scale);
#pragma unroll
  for (int e = 0; e < kAngles; ++e) {
    cosine[e] = 1.0F;
    sine[e] = 0.0F;
    int pair = 8 * lane + e;
    if (kLayout == kAnyHalves)
      pair = first + e < half ? first + e : first + e < a.rotary ? first + e - half : half;
    if (turns && head < turned_heads && pair < half && position >= 0)
      turn(scaled, a.inv_freq[pair], &cosine[e], &sine[e]);
  }
  for (; head < all_heads; head += step) {
    const int kind = head < a.heads ? 0 : head < turned_heads ? 1 : 2;
    const int of_kind = kind == 0 ? head : kind == 1 ? head - a.heads : head - turned_heads;
    uint16_t *dst;
    if (kind == 0) {
      dst = a.query + row * a.query_stride + static_cast<size_t>(head) * kDim;
    } else {
      if (page < 0)
        continue;
      dst = (kind == 1 ? a.cache.keys : a.cache.values) + at + of_kind * a.cache.head_stride;
    }
    float u[8], v[8];
    if (position < 0) {
      // A padding row's query.
#pragma unroll
      for (int e = 0; e < 8; ++e)
        u[e] = v[e] = 0.0F;
      store8<T>(dst + first, u);
      store8<T>(dst + second, v);
      continue;
    }
    const S *from = src + (a.column_split ? (of_kind * 3 + kind) * kDim : head * kDim);
    load8<S, kVector>(from + first, u);
    load8<S, kVector>(from + second, v);
    HeadSize size{1.0F, 1.0F};
    const float *weight = nullptr;
    if constexpr (kNormed) {
      if (kind != 2) {
        weight = kind == 0 ? norm.query_scale : norm.key_scale;
        if (weight != nullptr)
          weight += of_kind * norm.stride;
        float g[8], h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          g[e] = h[e] = 1.0F;
        if (weight != nullptr) {
          load8<float, true>(weight + first, g);
          load8<float, true>(weight + second, h);
        }
        size = head_size<kLanes>(u, v, norm);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[e] = u[e] * size.lift * size.inverse * g[e];
          v[e] = v[e] * size.lift * size.inverse * h[e];
        }
      }
    }
    if (kind == 2 || !turns) {
      store8<T>(dst + first, u);
      store8<T>(dst + second, v);
      continue;
    }
    float x[8], y[8];
    if (kLayout == kHalves) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = u[e] * cosine[e] - v[e] * sine[e];
        y[e] = v[e] * cosine[e] + u[e] * sine[e];
      }
    } else if (kLayout == kInterleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = u[2 * e] * cosine[e] - u[2 * e + 1] * sine[e];
        x[2 * e + 1] = u[2 * e + 1] * cosine[e] + u[2 * e] * sine[e];
        y[2 * e] = v[2 * e] * cosine[4 + e] - v[2 * e + 1] * sine[4 + e];
        y[2 * e + 1] = v[2 * e + 1] * cosine[4 + e] + v[2 * e] * sine[4 + e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = first + e;
        const float self = e < 8 ? u[e % 8] : v[e % 8];
        float other = 0.0F;
        if (d < a.rotary) {
          const int partner = d < half ? d + half : d - half;
          other = to_float(from[partner]);
          if constexpr (kNormed)
            other = other * size.lift * size.inverse *
                    (weight != nullptr ? weight[partner] : 1.0F);
        }
        const float turned = self * cosine[e % kAngles] +
                             (d < half ? -other : other) * sine[e % kAngles];
        (e < 8 ? x : y)[e % 8] = turned;
      }
    }
    if (kLayout != kHalves) {
      // Elements past the rotated ones, which cosine 1 and sine 0 would keep
      // but for one beside an infinity.
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = first + e < a.rotary ? x[e] : u[e];
        y[e] = second + e < a.rotary ? y[e] : v[e];
      }
    }
    store8<T>(dst + first, x);
    store8<T>(dst + second, y);
  }
}

struct Launch {
  bool vector;
  const HeadNorm *norm;
  unsigned blocks;
  hipStream_t stream;
};

template <typename S, typename T, int kDim, bool kVector, bool kNormed>
void launch_layout(const AppendArgs &a, const Launch &l) {
  auto kernel = paged_append_kernel<S, T, kDim, kVector, kAnyHalves, kNormed>;
  if (a.interleaved)
    kernel = paged_append_kernel<S, T, kDim, kVector, kInterleaved, kNormed>;
  else if (a.rotary % 16 == 0)
    kernel = paged_append_kernel<S, T, kDim, kVector, kHalves, kNormed>;
  hipLaunchKernelGGL(kernel, dim3(l.blocks), dim3(256), 0, l.stream, a,
                     kNormed ? *l.norm : HeadNorm{});
}

template <typename S, typename T, int kDim>
void launch_dim(const AppendArgs &a, const Launch &l) {
  if (l.norm == nullptr)
    return l.vector ? launch_layout<S, T, kDim, true, false>(a, l)
                    : launch_layout<S, T, kDim, false, false>(a, l);
  return l.vector ? launch_layout<S, T, kDim, true, true>(a, l)
                  : launch_layout<S, T, kDim, false, true>(a, l);
}

template <typename S, typename T> void launch_append(const AppendArgs &a, const Launch &l) {
  switch (a.cache.head_dim) {
  case 32:
    return launch_dim<S, T, 32>(a, l);
  case 64:
    return launch_dim<S, T, 64>(a, l);
  default:
    return launch_dim<S, T, 128>(a, l);
  }
}

template <typename S> void launch_source(const AppendArgs &a, const Launch &l) {
  if (a.cache.dtype == kElementBF16)
    launch_append<S, __bf16>(a, l);
  else
    launch_append<S, _Float16>(a, l);
}

}  // namespace

Status paged_append(const PagedCache &cache, const PagedBatch &batch, int dtype,
                    const void *projected, size_t row_stride, size_t heads, bool column_split,
                    const PagedRope &rope, void *query, size_t query_stride,
                    hipStream_t stream, const HeadNorm *norm) {
  const size_t kv = static_cast<size_t>(cache.kv_heads), dim = static_cast<size_t>(cache.head_dim);
  if (projected == nullptr || query == nullptr || heads == 0 || heads > (1U << 16) ||
      heads % kv != 0 || (column_split && heads != kv))
    return {ErrorCode::kInvalidArgument,
            "paged_append: null tensor, or heads that are no multiple of kv_heads"};
  if (dtype != kElementF32 && dtype != kElementBF16 && dtype != kElementF16)
    return {ErrorCode::kInvalidArgument, "paged_append: the projection is F32, BF16 or F16"};
  const size_t size = dtype == kElementF32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(projected) % size != 0 || row_stride < (heads + 2 * kv) * dim)
    return {ErrorCode::kInvalidArgument, "paged_append: row_stride below the row's width"};
  if (reinterpret_cast<uintptr_t>(query) % 16 != 0 || query_stride % 8 != 0 ||
      query_stride < heads * dim)
    return {ErrorCode::kInvalidArgument,
            "paged_append: query rows have to start on 16 bytes and hold every head"};
  if (rope.rotary_dim % 2 != 0 || rope.rotary_dim > dim ||
      (rope.rotary_dim != 0 &&
       (rope.inv_freq == nullptr || !(rope.scale > 0.0F) || !std::isfinite(rope.scale))))
    return {ErrorCode::kInvalidArgument, "paged_append: invalid rotation"};
  if (norm != nullptr &&
      ((reinterpret_cast<uintptr_t>(norm->query_scale) |
        reinterpret_cast<uintptr_t>(norm->key_scale)) % 16 != 0 ||
       norm->stride % 4 != 0 || (norm->stride != 0 && norm->stride < dim) ||
       norm->stride > (size_t{1} << 30) || !(norm->eps > 0.0F) || norm->eps > 1.0F))
    return {ErrorCode::kInvalidArgument,
            "paged_append: norm scales have to start on 16 bytes, eps is above 0 and at most 1"};
  const bool vector = reinterpret_cast<uintptr_t>(projected) % 16 == 0 &&
                      row_stride * size % 16 == 0;
  // A block's pass over the heads; few rows are split over them. us split and whole, 32
  // heads of each kind: 1 row 4.3 and 4.7, 27 rows 5.5 and 6.1, 103 rows 6.3 and 6.6, 264
  // rows 8.2 and 8.0, 428 rows 10.5 and 9.5.
  const size_t passes = ceil_div((heads + 2 * kv) * (dim / 16), 256);
  const size_t parts = batch.tokens > 128 ? 1 : passes;
  const size_t blocks = parts * static_cast<size_t>(batch.tokens);
  if (blocks > ((size_t{1} << 32) - 1) / 256)  // a launch counts its threads in 32 bits
    return {ErrorCode::kInvalidArgument, "paged_append: grid too large"};
  const AppendArgs args{cache, batch, projected, row_stride, static_cast<int>(heads),
                        column_split ? 1 : 0, rope.inv_freq, static_cast<int>(rope.rotary_dim),
                        rope.interleaved ? 1 : 0, rope.rotary_dim != 0 ? rope.scale : 1.0F,
                        static_cast<uint16_t *>(query), query_stride, static_cast<int>(parts)};
  const Launch launch{vector, norm, static_cast<unsigned>(blocks), stream};
  if (dtype == kElementF32)
    launch_source<float>(args, launch);
  else if (dtype == kElementBF16)
    launch_source<__bf16>(args, launch);
  else
    launch_source<_Float16>(args, launch);
  return launch_status("paged_append_kernel");
}

}  // namespace evo::hip
