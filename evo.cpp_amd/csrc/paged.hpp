// SPDX-License-Identifier: Apache-2.0
// The paged cache and the rows of a batch, as the kernels see them, and the
// index rules that every kernel over them goes by. The device arrays hold what
// the caller wrote there, so each rule bounds what it returns: no entry leads
// outside the tensors. Host code too, for the tests.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace evo::hip {

struct PagedCache {
  int dtype;  // ElementType: BF16 or F16
  uint16_t *keys, *values;
  int pages;
  int page_shift;  // log2 of the page size
  int kv_heads, head_dim;
  size_t page_stride, head_stride, token_stride;  // elements
};

struct PagedBatch {
  int sequences, tokens, max_tokens, max_length;
  const int32_t *token_start, *lengths, *page_table;
  size_t table_stride;
  int shared_length;
  const int32_t *shared_table;
  int32_t *error;
};
constexpr int kBadSequence = 1, kBadPage = 2;

// Rows [first, first + count) of a sequence, at positions length - count ..
// length - 1 (negative: padding).
struct SequenceRows {
  int first, count, length;
  bool valid;
};
__host__ __device__ inline SequenceRows sequence_rows(const PagedBatch &batch, int sequence) {
  SequenceRows rows{batch.token_start[sequence], 0, batch.lengths[sequence], false};
  const int end = batch.token_start[sequence + 1];
  // (Order and range first: the difference of two arbitrary words overflows.)
  if (rows.first < 0 || end < rows.first || end > batch.tokens ||
      end - rows.first > batch.max_tokens || rows.length < 0 || rows.length > batch.max_length)
    return rows;
  rows.count = end - rows.first;
  // Rows on shared positions: there is no such row (length 0: padding only).
  if (batch.shared_length > 0 && rows.count > 0 && rows.length != 0 &&
      rows.length - rows.count < batch.shared_length)
    return rows;
  rows.valid = true;
  return rows;
}

// The sequence that owns row `token`, or -1. token_start is searched as if it
// ascended; the answer is checked, so an unordered array gives -1 at worst.
__host__ __device__ inline int sequence_of(const PagedBatch &batch, int token) {
  // Row i of sequence i: a decode step.
  const int same = token < 0 ? 0 : token < batch.sequences ? token : batch.sequences - 1;
  if (batch.token_start[same] <= token && token < batch.token_start[same + 1])
    return same;
  int low = 0, high = batch.sequences;  // the answer lies in [low, high)
  while (high - low > 1) {
    const int middle = low + (high - low) / 2;
    if (batch.token_start[middle] <= token)
      low = middle;
    else
      high = middle;
  }
  return batch.token_start[low] <= token && token < batch.token_start[low + 1] ? low : -1;
}

// Page of table entry `index`, or -1 where it holds none.
__host__ __device__ inline int checked_page(const int32_t *table, int index, int pages) {
  const int page = table[index];
  return page >= 0 && page < pages ? page : -1;
}

#if defined(__HIPCC__)
__device__ inline void report(const PagedBatch &batch, int bit) {
  if (batch.error != nullptr)
    atomicOr(batch.error, bit);
}
// One block of a launch looks all sequences over.
__device__ inline void report_bad_sequences(const PagedBatch &batch) {
  if (batch.error == nullptr)
    return;
  for (int i = threadIdx.x; i < batch.sequences; i += blockDim.x)
    if (!sequence_rows(batch, i).valid)
      report(batch, kBadSequence);
}
#endif

}  // namespace evo::hip
