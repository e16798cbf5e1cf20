// SPDX-License-Identifier: Apache-2.0
// Reductions and scans over the lanes of a wave and the waves of a block, and the
// order of logits: what the kernels over rows of logits share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace evo::hip {

// Order of the values as integers; -0 and 0 are one value.
__device__ inline uint32_t ordered(float v) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0F);
  return (bits & 0x80000000U) != 0 ? ~bits : bits | 0x80000000U;
}

struct Most {
  template <typename V> __device__ V operator()(V x, V y) const { return x > y ? x : y; }
  template <typename V> static __device__ V identity() {
    return std::is_same_v<V, float> ? static_cast<V>(-INFINITY) : static_cast<V>(0);
  }
};
struct Least {
  template <typename V> __device__ V operator()(V x, V y) const { return x < y ? x : y; }
  template <typename V> static __device__ V identity() {
    return std::is_same_v<V, float> ? static_cast<V>(INFINITY)
           : std::is_same_v<V, int> ? static_cast<V>(0x7fffffff)
                                    : static_cast<V>(~0ULL);
  }
};
struct Sum {
  template <typename V> __device__ V operator()(V x, V y) const { return x + y; }
  template <typename V> static __device__ V identity() { return 0; }
};

// v of another lane, by the DPP control kCtrl; `other` in lanes it has none for.
template <int kCtrl, int kRows, typename V> __device__ inline V dpp(V other, V v) {
  constexpr int kWords = sizeof(V) / 4;
  uint32_t from[kWords], to[kWords];
  __builtin_memcpy(from, &v, sizeof(V));
  __builtin_memcpy(to, &other, sizeof(V));
#pragma unroll
  for (int i = 0; i < kWords; ++i)
    to[i] = __builtin_amdgcn_update_dpp(to[i], from[i], kCtrl, kRows, 0xf, false);
  __builtin_memcpy(&v, to, sizeof(V));
  return v;
}
// f over the lanes 0 .. this one: rows of 16 lanes, then row to row, in registers
// (shuffles go through LDS: six of them take a microsecond of a lone wave).
template <typename F, typename V> __device__ inline V wave_scan(V v) {
  const F f;
  const V none = F::template identity<V>();
  v = f(v, dpp<0x111, 0xf>(none, v));  // row_shr 1, 2, 4, 8
  v = f(v, dpp<0x112, 0xf>(none, v));
  v = f(v, dpp<0x114, 0xf>(none, v));
  v = f(v, dpp<0x118, 0xf>(none, v));
  v = f(v, dpp<0x142, 0xa>(none, v));  // row_bcast 15: into rows 1 and 3
  return f(v, dpp<0x143, 0xc>(none, v));  // row_bcast 31: into rows 2 and 3
}
template <typename V> __device__ inline V lane_value(V v, int lane) {
  constexpr int kWords = sizeof(V) / 4;
  uint32_t words[kWords];
  __builtin_memcpy(words, &v, sizeof(V));
#pragma unroll
  for (int i = 0; i < kWords; ++i)
    words[i] = __builtin_amdgcn_readlane(words[i], lane);
  __builtin_memcpy(&v, words, sizeof(V));
  return v;
}
template <typename V, typename F> __device__ inline V wave_reduce(V v, F) {
  return lane_value(wave_scan<F>(v), 63);
}
template <int kThreads, typename V, typename F>
__device__ inline V block_reduce(V v, V *scratch, F f) {
  v = wave_reduce(v, f);
  if constexpr (kThreads > 64) {
    const int lane = threadIdx.x & 63;
    __syncthreads();
    if (lane == 0)
      scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave_reduce(lane < kThreads / 64 ? scratch[lane] : F::template identity<V>(), f);
  }
  return v;
}

// Between a wave's own writes to LDS and its reads of them.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace evo::hip
