/* SPDX-License-Identifier: Apache-2.0
 *
 * Operator-level C ABI of libevo_hip.so: the gfx950 kernels of the
 * StripedHyena2 prefill path on caller-owned device memory.
 *
 * All pointers are device pointers (hipMalloc'd or a torch tensor's
 * data_ptr()); `stream` is a hipStream_t (NULL = the default stream). Calls
 * are asynchronous on that stream and never allocate device memory: every
 * temporary lives in a caller-provided workspace whose size the matching
 * *_workspace_bytes query returns. Shapes are validated on the host before
 * any launch; invalid arguments return EVO_STATUS_INVALID_ARGUMENT with the
 * message in evo_last_error(). BF16 tensors are raw uint16 bit patterns.
 *
 * Each entry point names the reference interface it replaces.
 */
#ifndef EVO_HIP_OPS_H
#define EVO_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "evo/evo.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Whole-sequence prefill with tokens (uint32 [count]) and logits (F32
 * [count, vocab]) in device memory, for callers that keep the stream on the
 * GPU (serving loops, benchmarks): same chunk loop, caches and numerics as
 * evo_context_prefill, but no host copies; synchronises the context stream
 * once at the end. The context is reset first (position 0), so one context can
 * serve successive sequences. Token ids >= vocab fail the call.
 * Replaces the CUDA `PipelineModel::prefill` loop driven from
 * `src/c_api.cpp:962-989`, minus the host logits. */
EVO_API evo_status evo_hip_context_prefill_resident(evo_context *context,
                                                    const uint32_t *tokens,
                                                    size_t count, float *logits);
/* The context's HIP stream (hipStream_t), for ordering caller work. */
EVO_API void *evo_hip_context_stream(const evo_context *context);

/* Measurement hooks (no counterpart in the reference): with timing on, each
 * prefill records HIP events on the context stream around every layer's MLP
 * l1/l2 product (the dominant kernel); evo_hip_context_product_time returns
 * the summed duration (ms) and the number of launches of the last chunk
 * prefilled, once the caller has seen that prefill complete. Off by default. */
EVO_API evo_status evo_hip_context_set_product_timing(evo_context *context, int enable);
EVO_API evo_status evo_hip_context_product_time(const evo_context *context, float *ms,
                                                size_t *launches);

/* Storage type of activation tensors passed to the Hyena operator. */
/* EVO_HIP_SPLIT: F32 input, output as split BF16 planes [2][rows][cols]
 * (hi = bf16(y), lo = bf16(y - hi)), the GEMM activation layout.
 * EVO_HIP_BF16_SPLIT: BF16 input (the FP8 projection's output), split
 * output; Hyena operator only.
 * EVO_HIP_F16 / EVO_HIP_BF16_F16: F32 / BF16 input, output one FP16 plane
 * [rows][cols], fp16(y) rounded to nearest even and saturated to +-65504
 * (the activation of the one-pass FP16 out-projection); Hyena operator
 * only. */
typedef enum evo_hip_dtype {
  EVO_HIP_F32 = 0,
  EVO_HIP_BF16 = 1,
  EVO_HIP_SPLIT = 2,
  EVO_HIP_BF16_SPLIT = 3,
  EVO_HIP_F16 = 4,
  EVO_HIP_BF16_F16 = 5,
  /* OR-ed into the Hyena operator's dtype: the projection holds stream s
   * (x2, x1, v) of channel c at column s*W + c instead of the reference's
   * 3c + s (the library permutes its projection weights this way). */
  EVO_HIP_PLANAR = 0x100,
  /* OR-ed into the Hyena operator's dtype: every inner_filter tap is a BF16
   * value (evo2 artifacts store `filter.h` as BF16), which lets the HCM
   * operator form its Toeplitz product in two MFMA passes instead of three
   * (same result). */
  EVO_HIP_BF16_TAPS = 0x200
} evo_hip_dtype;
typedef enum evo_hip_hyena_kind {
  EVO_HIP_HYENA_HCS = 0,
  EVO_HIP_HYENA_HCM = 1,
  EVO_HIP_HYENA_HCL = 2
} evo_hip_hyena_kind;

/* Fused Hyena mixer of one block: short FIR (short_len taps, per column of
 * the [L, 3W] projection with interleaved (x2, x1, v) triples), u = x1*v, the
 * long filter (HCS grouped FIR / HCM grouped causal conv + D*u / HCL modal
 * recurrence + D*u), times x2; output [L, W] in `dtype`.
 * Replaces evo.cpp `bf16_fir_prefill_direct` + `bf16_hcs_prefill` /
 * `bf16_hcm_prefill` / `bf16_hcl_prefill`
 * (`include/evo/cuda/hyena.hpp:154-252`) and the CPU mixer
 * (`src/cpu/model.cpp:546-605`).
 *   short_filter  BF16 [3W, short_len]
 *   inner_filter  F32 [groups, inner_len]          (HCS/HCM; else NULL)
 *   direct        F32 [W]                          (HCM/HCL; else NULL)
 *   poles         F32 [W, state] = exp(log_poles)  (HCL; else NULL)
 *   residues      F32 [W, state]                   (HCL; else NULL)
 *   short_history F32 [short_len-1, 3W], inner_history F32 [inner_len-1, W],
 *   modal_state   F32 [W, state]: optional continuation caches (NULL = zero
 *                 initial state, nothing kept); read as the state before row
 *                 0 and overwritten with the state after row L-1. */
EVO_API size_t evo_hip_hyena_workspace_bytes(evo_hip_hyena_kind kind,
                                             size_t length, size_t width,
                                             size_t state_size);
EVO_API evo_status evo_hip_hyena_forward(
    evo_hip_hyena_kind kind, evo_hip_dtype dtype, const void *projection,
    size_t length, size_t width, const uint16_t *short_filter,
    size_t short_len, const float *inner_filter, size_t groups,
    size_t inner_len, const float *direct, const float *poles,
    const float *residues, size_t state_size, float *short_history,
    float *inner_history, float *modal_state, void *workspace,
    size_t workspace_bytes, void *output, void *stream);

/* Allocation-free variant of evo_hip_hyena_forward: same arguments minus
 * the workspace, same kernels and results. The workspace comes from a fixed
 * device array of evo_hip_hyena_static_scratch_bytes() (32 MiB) in the
 * library, one per device, held until the process ends; the call fails with
 * EVO_STATUS_INVALID_ARGUMENT, before any launch, when the path the shape
 * takes keeps more than that in its workspace. Only two paths use one: the
 * three-pass HCL fallback (planar projections, short filters other than 3
 * taps, W % 16 != 0; chunk states of evo_hip_hyena_workspace_bytes()) and
 * the F32-tap HCS/HCM MFMA FIR (its Toeplitz table, 2.6 MB at W = 4096).
 * The model's shapes (one-pass HCL, streaming HCS/HCM) need none and are
 * accepted at any length.
 * The call makes no device allocation (no hipMalloc/hipFree), so callers that
 * cannot allocate (code under HIP graph capture, tight serving loops) can
 * use it. Every call on a device shares that device's array: calls that
 * overlap on one device (different streams, threads) race; serialise them.
 * No counterpart in the reference: evo.cpp's operators always receive their
 * scratch from the caller or allocate it. */
EVO_API size_t evo_hip_hyena_static_scratch_bytes(void);
EVO_API evo_status evo_hip_hyena_forward_static(
    evo_hip_hyena_kind kind, evo_hip_dtype dtype, const void *projection,
    size_t length, size_t width, const uint16_t *short_filter,
    size_t short_len, const float *inner_filter, size_t groups,
    size_t inner_len, const float *direct, const float *poles,
    const float *residues, size_t state_size, float *short_history,
    float *inner_history, float *modal_state, void *output, void *stream);

/* codes[i] = E4M3FN(float(bf16(x[i])) * scale), RNE, satfinite.
 * Replaces `software_e4m3_quantize_bf16_codes` (`include/evo/cuda/ops.hpp:92-96`). */
EVO_API evo_status evo_hip_e4m3_quantize(evo_hip_dtype dtype, const void *x,
                                         size_t count, float scale,
                                         uint8_t *codes, void *stream);

/* Software-FP8 projection out[M,N] = bf16(QGMMA(in_codes[M,K], w_codes[N,K])
 * * output_scale), stored as F32. mode 0 = E4M3 MFMA with promotion every 32
 * K, 1 = every 128 K, 2 = bit-exact integer QGMMA emulation.
 * Replaces `software_e4m3_h100_linear` (`include/evo/cuda/ops.hpp:104-114`). */
EVO_API evo_status evo_hip_fp8_linear(const uint8_t *in_codes,
                                      const uint8_t *w_codes, float *out,
                                      size_t m, size_t n, size_t k,
                                      float output_scale, int mode,
                                      void *stream);

/* The same product stored as BF16 [M,N] (the projection's own output type:
 * each value already is bf16(acc * output_scale)). */
EVO_API evo_status evo_hip_fp8_linear_bf16(const uint8_t *in_codes,
                                           const uint8_t *w_codes, uint16_t *out,
                                           size_t m, size_t n, size_t k,
                                           float output_scale, int mode, void *stream);

/* GEMM activation layout: hi[i] = bf16(x[i]), lo[i] = bf16(x[i] - hi[i])
 * (lo may be NULL for BF16-only activations). */
EVO_API evo_status evo_hip_split_f32(const float *x, size_t count, uint16_t *hi,
                                     uint16_t *lo, void *stream);

/* out[M,N] = x[M,K] . w[N,K]^T (+ bf16 bias[N]) (+ residual[M,N]); x as
 * split BF16 planes (x_lo NULL: one BF16 MFMA pass), w BF16, out F32.
 * Replaces `bf16_linear` (`include/evo/cuda/ops.hpp:61-70`) and the CPU
 * `linear` (`src/cpu/model.cpp:284-314`). */
EVO_API evo_status evo_hip_linear(const uint16_t *x_hi, const uint16_t *x_lo,
                                  const uint16_t *w, const uint16_t *bias,
                                  const float *residual, size_t m, size_t n,
                                  size_t k, float *out, void *stream);

/* evo_hip_linear with an F32 device workspace (16-byte aligned; otherwise
 * it is not used): launches with few output tiles split K across blocks
 * (partials in the workspace, summed in split order before the epilogue),
 * the path the model takes for short prompts. The same reference interface
 * as evo_hip_linear. */
EVO_API evo_status evo_hip_linear_split(const uint16_t *x_hi, const uint16_t *x_lo,
                                        const uint16_t *w, const uint16_t *bias,
                                        const float *residual, size_t m, size_t n,
                                        size_t k, float *out, float *workspace,
                                        size_t workspace_bytes, void *stream);

/* Gated MLP out[M,W] = l3(act(l1 x) * l2 x) (+ residual) with act = erf-GELU
 * when gelu != 0. w12 is the interleaved [2*Fp, W] l1/l2 weight (32-row
 * blocks, Fp = F rounded up to 32) built by evo_hip_pack_mlp;
 * inner_workspace holds the gated [M, F] activation as split planes
 * (2*M*F uint16, or M*F when x_lo is NULL).
 * Replaces `bf16_mlp` (`include/evo/cuda/ops.hpp:133-138`). */
EVO_API evo_status evo_hip_pack_mlp(const uint16_t *l1, const uint16_t *l2,
                                    size_t inner, size_t width, uint16_t *w12,
                                    void *stream);
EVO_API evo_status evo_hip_gated_mlp(const uint16_t *x_hi, const uint16_t *x_lo,
                                     const uint16_t *w12, const uint16_t *l3,
                                     size_t m, size_t width, size_t inner,
                                     int gelu, uint16_t *inner_workspace,
                                     const float *residual, float *out,
                                     void *stream);

/* RMSNorm y = x / (sqrt(mean(x^2)) + eps) * scale over rows of width,
 * written as F32 (out) and/or split BF16 planes (out_hi, out_lo).
 * Replaces `bf16_rms_norm` (`include/evo/cuda/ops.hpp:117-120`). */
EVO_API evo_status evo_hip_rms_norm(const float *x, size_t rows, size_t width,
                                    const float *scale, float eps, float *out,
                                    uint16_t *out_hi, uint16_t *out_lo,
                                    void *stream);

/* RMSNorm fused with the FP8 projection's input quantisation: codes =
 * E4M3FN(bf16(y) * code_scale) of the normed rows, without writing y
 * (the sequence `bf16_rms_norm` + `quantize_bf16_e4m3` of the reference's
 * FP8 projection path, `src/cuda/ops.cu:72-113, 250-262`). */
EVO_API evo_status evo_hip_rms_norm_e4m3(const float *x, size_t rows, size_t width,
                                         const float *scale, float eps, float code_scale,
                                         uint8_t *codes, void *stream);

/* Few-row products (m <= 4, the decode step) of RMSNorm'd rows without the
 * norm's own launch: each block normalises x [m, k] (F32, 16-byte aligned,
 * scale [k]) itself in the order evo_hip_rms_norm uses, so the results equal
 * evo_hip_rms_norm (split planes when split != 0, else hi only) followed by
 * evo_hip_linear, and evo_hip_rms_norm_e4m3 followed by
 * evo_hip_fp8_linear_bf16 (modes 0 and 1), bit for bit. They fuse the
 * reference's `bf16_rms_norm` with `bf16_linear` / the FP8 projection
 * (`include/evo/cuda/ops.hpp:61-70, 104-120`) for the decode path. */
EVO_API evo_status evo_hip_linear_normed(const float *x, size_t m, size_t k,
                                         const float *scale, float eps, int split,
                                         const uint16_t *w, size_t n, float *out,
                                         void *stream);
EVO_API evo_status evo_hip_fp8_linear_normed(const float *x, size_t m, size_t k,
                                             const float *scale, float eps,
                                             float input_scale, const uint8_t *w_codes,
                                             size_t n, float output_scale, int mode,
                                             uint16_t *out, void *stream);

/* Attention block body: split the Wqkv output [rows, 3W], apply RoPE at
 * positions prefix.., append K/V at `prefix` of the caches, causal softmax
 * attention into out [rows, W] F32. query is workspace of 2*rows*W uint16;
 * key_cache holds split BF16 planes [2][capacity][W] uint16 and value_cache
 * the transposed planes [2][W][capacity], each 16-position block stored in
 * the order 0-3, 8-11, 4-7, 12-15. capacity must be a multiple of 64, and
 * cache entries never written must hold finite values (zero the caches once).
 * Replaces `bf16_split_qkv` + `bf16_apply_rope` + `bf16_kv_append` +
 * `bf16_online_causal_attention` (`include/evo/cuda/attention.hpp:100-133`). */
EVO_API evo_status evo_hip_attention(const float *projected, size_t rows,
                                     size_t width, size_t heads,
                                     int column_split, const float *inv_freq,
                                     float rope_scale, size_t prefix,
                                     uint16_t *query, uint16_t *key_cache,
                                     uint16_t *value_cache, size_t capacity,
                                     float *out, void *stream);

/* evo_hip_attention with an F32 device workspace, the decode step's path:
 * - A single query (rows == 1, head_dim 32/64/128) is split over its keys if
 *   the workspace holds a part (max, sum and head_dim outputs: head_dim + 2
 *   floats) per head and 256 keys. Chunks are whole 64-key tiles: one each
 *   below 4096 blocks (tiles x heads) and up to 512 chunks, more beyond that,
 *   and at least four where the workspace holds no more parts (32 heads: 64
 *   keys per chunk at 4096 keys, 512 at 32768, 2048 at 131072).
 * - A few rows, or the last rows of a prompt, are split over parts of their
 *   keys where that is faster and the workspace holds the parts (rows, rounded
 *   up to 128 or 256, x heads x parts x (head_dim + 2) floats).
 * The same reference interface. */
EVO_API evo_status evo_hip_attention_ws(const float *projected, size_t rows,
                                        size_t width, size_t heads,
                                        int column_split, const float *inv_freq,
                                        float rope_scale, size_t prefix,
                                        uint16_t *query, uint16_t *key_cache,
                                        uint16_t *value_cache, size_t capacity,
                                        float *out, float *workspace,
                                        size_t workspace_bytes, void *stream);

/* ---- Several sequences at a time: a paged key/value cache, the attention
 * that reads it, and sampling. No counterpart in the reference, whose batch
 * size is one.
 *
 * A paged cache holds the keys and values of any number of sequences in pages
 * of page_size positions that the caller hands out. Position p of a sequence
 * lies in page page_table[sequence][p / page_size], slot p % page_size; the
 * element d of key/value head h there is at
 *   pages + page * page_stride + h * head_stride + slot * token_stride + d.
 * dtype: EVO_HIP_BF16 or EVO_HIP_F16. page_size: a power of two from 16 to
 * 32768. head_dim: 32, 64 or 128. The strides count elements and are
 * multiples of 8, token_stride at most 2^24; all three 0 means dense
 * [pages][kv_heads][page_size][head_dim]. Both bases are 16-byte aligned. Slots that no
 * sequence has written may hold anything. */
typedef struct evo_hip_paged_cache {
  size_t struct_size;
  evo_hip_dtype dtype;
  void *key_pages;
  void *value_pages;
  size_t pages;
  size_t page_size;
  size_t kv_heads;
  size_t head_dim;
  size_t page_stride;
  size_t head_stride;
  size_t token_stride;
} evo_hip_paged_cache;

/* The rows of one call: `tokens` rows of a projection, query or output, of
 * which sequence s has the rows token_start[s] .. token_start[s + 1] - 1, its
 * newest tokens. lengths[s] counts its positions, these tokens included, so
 * its last row is at position lengths[s] - 1. Where it has more rows than
 * positions, the first ones are padding. Rows behind the last sequence's
 * (token_start[sequences] < tokens) belong to none and are left as they are.
 *   max_tokens, max_length: host bounds on a sequence's rows and positions
 *     (max_length <= table_stride * page_size, at most 2^30). They choose the
 *     launches: close bounds run faster. tokens is at most 2^24, sequences at
 *     most 2^20, and a launch 2^24 blocks: a call that would need more is refused
 *     (attention takes a block for each key/value head of each sequence and of each
 *     16 or 128 rows, times the chunks of its keys; tokens * heads is below 2^31 - 128).
 *   token_start, lengths, page_table: int32 device arrays, read by each call
 *     when it runs, so a captured graph follows their changes within the
 *     bounds; page_table [sequences][table_stride].
 *   shared_length: positions at the beginning that all sequences share, a
 *     multiple of page_size (0: none), in the pages of the device array
 *     shared_table (shared_length / page_size entries). Entries of page_table
 *     for these positions are not read. Every sequence with rows has
 *     lengths[s] == 0 or its rows behind the shared positions.
 *   error: optional device word; the kernels OR the bits below into it and
 *     never clear it.
 * The device arrays cannot be checked on the host. A sequence whose entries
 * break these rules (bounds, order, shared positions) is left out, its rows
 * left as they are: EVO_HIP_PAGED_BAD_SEQUENCE. A page index outside
 * [0, pages) that a call needs is never followed: nothing is written there,
 * and its positions count as masked: EVO_HIP_PAGED_BAD_PAGE. */
typedef struct evo_hip_paged_batch {
  size_t struct_size;
  size_t sequences;
  size_t tokens;
  size_t max_tokens;
  size_t max_length;
  const int32_t *token_start;
  const int32_t *lengths;
  const int32_t *page_table;
  size_t table_stride;
  size_t shared_length;
  const int32_t *shared_table;
  int32_t *error;
} evo_hip_paged_batch;
#define EVO_HIP_PAGED_BAD_SEQUENCE 1
#define EVO_HIP_PAGED_BAD_PAGE 2

/* Splits the QKV projection of a batch's rows, rotates queries and keys by
 * their positions, and appends keys and values to the cache in the same pass.
 *   projected  [tokens][row_stride] F32, BF16 or F16 (dtype); columns
 *              [query heads | key heads | value heads][head_dim], or with
 *              column_split [head][query, key, value][head_dim] (heads ==
 *              kv_heads). heads is a multiple of kv_heads.
 *   rotation   of the first rotary_dim elements (even, 0: none) of each query
 *              and key head, by the angle (position / rope_scale) *
 *              inv_freq[i] (F32 [rotary_dim / 2]), formed in 64 bits so that far
 *              positions keep their angle. Pair i is (i, rotary_dim / 2 + i),
 *              or (2i, 2i + 1) when interleaved.
 *   query      [tokens][query_stride] in the cache's dtype, the rotated
 *              queries (rows of 16-byte aligned heads, query_stride a multiple
 *              of 8); padding rows are zeroed and append nothing.
 * Rounded once, to nearest even; a value beyond FP16 becomes infinity. query
 * must not overlap projected, and two sequences must not append to one slot. */
EVO_API evo_status evo_hip_paged_append(const evo_hip_paged_cache *cache,
                                        const evo_hip_paged_batch *batch,
                                        evo_hip_dtype dtype, const void *projected,
                                        size_t row_stride, size_t heads, int column_split,
                                        const float *inv_freq, size_t rotary_dim,
                                        int interleaved, float rope_scale, void *query,
                                        size_t query_stride, void *stream);

/* evo_hip_paged_append of query and key heads that are normalized before they are
 * rotated, each by its own root mean square over head_dim:
 *   y = x / (sqrt(mean(x^2)) + eps) * scale           (as evo_hip_rms_norm), or
 *   y = x / sqrt(mean(x^2) + eps) * scale             with eps_inside.
 * Values are stored as they are. Formed in F32 (a head whose squares would leave its
 * range is brought near one first) and rounded once, after the rotation; a head that
 * holds an infinity becomes what the formula gives: NaN there, zero elsewhere.
 *   query_scale, key_scale  F32 [head_dim], one for all heads (scale_stride 0) or
 *              [heads], [kv_heads][scale_stride] (a multiple of 4, head_dim at least);
 *              16-byte aligned; NULL: 1.
 *   eps        above 0, at most 1.
 * The other arguments, and what they refuse, are evo_hip_paged_append's. */
EVO_API evo_status evo_hip_paged_append_normed(
    const evo_hip_paged_cache *cache, const evo_hip_paged_batch *batch, evo_hip_dtype dtype,
    const void *projected, size_t row_stride, size_t heads, int column_split,
    const float *query_scale, const float *key_scale, size_t scale_stride, float eps,
    int eps_inside, const float *inv_freq, size_t rotary_dim, int interleaved, float rope_scale,
    void *query, size_t query_stride, void *stream);

/* Attention of a batch's rows over the cache: for each row and query head h
 *   out = sum_k softmax_k(scale * query . key[k]) * value[k]
 * over the positions k up to the row's own, of key/value head
 * h / (heads / kv_heads); a row that sees none (padding, length 0) is zero.
 * The rows' own keys are in the cache already (evo_hip_paged_append).
 *   query  [tokens][query_stride] and out [tokens][out_stride], the cache's
 *          dtype, heads side by side, 16-byte aligned, strides multiples of 8;
 *          out may be query, with the same stride.
 *   scale  positive and below 2.3e38 (1 / sqrt(head_dim) as a rule).
 * With shared_length the prefix's keys are read once for the rows of all
 * sequences, not once for each.
 * What a row does not see has no effect on it, infinities and NaN included:
 * positions behind its own, slots behind a sequence's length, other pages, other rows.
 * Scores and sums are F32. Weights are rounded to the cache's type for their product
 * with the values: BF16 to 2^-8 of each, FP16 to 2^-11 of each that is at least 2^-23
 * of the row's largest, the others to 2^-34 of the largest. A row whose every score is
 * -infinity is zero.
 * The workspace (16-byte aligned, no initial contents) takes the partial
 * results of keys that are split over blocks; its size depends on the host
 * fields of the structs and heads alone. It does not grow with the batch (few
 * rows are split more), but two phases (own keys, shared ones) take at most
 * 136 MB each, or tokens * heads * (head_dim + 2) * 4 bytes where that is more.
 * Calls that overlap need one each. */
EVO_API size_t evo_hip_paged_attention_workspace_bytes(const evo_hip_paged_cache *cache,
                                                       const evo_hip_paged_batch *batch,
                                                       size_t heads);
EVO_API evo_status evo_hip_paged_attention(const evo_hip_paged_cache *cache,
                                           const evo_hip_paged_batch *batch,
                                           const void *query, size_t query_stride,
                                           size_t heads, float scale, void *out,
                                           size_t out_stride, void *workspace,
                                           size_t workspace_bytes, void *stream);

/* tokens[r] = one token of row r of logits [rows][row_stride] (F32, BF16 or
 * F16; rows and vocab at most 2^20), in the order and with the cuts of evo_sampler_sample:
 * tokens by descending logit, equal ones by ascending index; of these the first
 * top_k (0, or vocab and more: all); weights exp(logit / temperature) in 64 bits,
 * held to 2^-(B+1) of the largest, B = 63 - ceil(log2(vocab)) and 51 at most (one
 * below that counts as none, and a border is off by vocab times that at most);
 * of these the shortest beginning whose weight reaches top_p of what top-k left
 * (1: all); of these the ones of at least min_p times the largest weight (0: all);
 * then the first whose cumulative weight exceeds uniform times the weight left.
 * temperature 0, or top_k 1: the first token.
 *   temperature, top_p, min_p (F32), top_k (int32): device [rows], or NULL for
 *     1, 1, 0 and 0.
 *   uniform: device F32 [rows], in [0, 1) (beyond: its nearer end). Its 24 bits are
 *     the draw's resolution: evo_sampler_sample draws 53, so the two agree where
 *     no border lies between its draw and the F32 one, and tokens of less than 2^-24
 *     of the weight are met in steps of that.
 * The device arrays are read when the call runs. A row gets UINT32_MAX where its
 * logits hold NaN or +infinity or nothing above -infinity, or its parameters are
 * out of range (temperature negative or not finite, top_k negative, top_p outside
 * (0, 1], min_p outside [0, 1], any NaN). The token does not depend on the
 * order in which the GPU works.
 * The workspace (16-byte aligned, no initial contents) lets few rows of a large
 * vocabulary be split over blocks; NULL: a block takes a whole row. Calls that
 * overlap need one each. */
EVO_API size_t evo_hip_sample_workspace_bytes(size_t rows, size_t vocab);
EVO_API evo_status evo_hip_sample(evo_hip_dtype dtype, const void *logits, size_t rows,
                                  size_t vocab, size_t row_stride, const float *temperature,
                                  const int32_t *top_k, const float *top_p,
                                  const float *min_p, const float *uniform,
                                  uint32_t *tokens, void *workspace,
                                  size_t workspace_bytes, void *stream);

/* Low-rank adapters, each a pair of BF16 matrices: down [rank][in_width] and up
 * [out_width][rank], `adapters` (at most 8192) of them behind each other.
 *   rank     rows of down and columns of up as they are stored, a multiple of 8 up to
 *            128; ranks (device int32 [adapters], or NULL: all `rank`) says how many of
 *            them each adapter has, 0 to rank. What lies behind those is not used.
 *   in_width a multiple of 8; both widths at most 2^24.
 *   down, up 16-byte aligned; down_stride, up_stride: elements from one adapter to the
 *            next, multiples of 8 (0: dense).
 *   scales   F32 [adapters], or NULL: 1.
 *   error    optional device word; EVO_HIP_BAD_ADAPTER is OR-ed into it, never cleared. */
typedef struct evo_hip_adapters {
  size_t struct_size;
  size_t adapters;
  size_t rank;
  size_t in_width;
  size_t out_width;
  const uint16_t *down;
  const uint16_t *up;
  size_t down_stride;
  size_t up_stride;
  const float *scales;
  const int32_t *ranks;
  int32_t *error;
} evo_hip_adapters;
#define EVO_HIP_BAD_ADAPTER 1

/* out[t] = residual[t] + scale_a * up_a . (down_a . x[t]) with a = adapter[t], the adapter of
 * row t of a batch, beside a product that all rows share (residual: what evo_hip_linear
 * wrote, its bias included, or NULL: zero).
 *   adapter  device int32 [rows], read when the call runs; -1: none, the row is its
 *            residual. An index or a rank outside the pool counts as none:
 *            EVO_HIP_BAD_ADAPTER. Rows may share adapters in any order.
 *   x        split BF16 planes [rows][x_stride] as evo_hip_linear takes them (x_lo NULL:
 *            one plane), 16-byte aligned, x_stride a multiple of 8; rows at most 2^20,
 *            both strides at most 2^40.
 *   residual, out  F32 [rows][out_stride], 4-byte aligned; out may be residual. Columns
 *            behind out_width are left as they are, so the columns of one projection may
 *            have adapters of their own. Whole 16 bytes of columns run faster.
 * Sums are F32; the inner values keep all of their 24 bits. An infinity or NaN in x or an
 * adapter reaches only the rows that use it; an infinity in up makes its column of those
 * infinite or NaN, which of both the call's sizes decide. Repeated calls give the same bits.
 * The workspace (16-byte aligned, no initial contents) holds the rows' order and the inner
 * values; calls that overlap need one each. One of the size for some rows serves calls of
 * fewer rows on the same pool too. */
EVO_API size_t evo_hip_adapter_linear_workspace_bytes(const evo_hip_adapters *pool, size_t rows);
EVO_API evo_status evo_hip_adapter_linear(const evo_hip_adapters *pool, const int32_t *adapter,
                                          const uint16_t *x_hi, const uint16_t *x_lo,
                                          size_t x_stride, size_t rows, const float *residual,
                                          float *out, size_t out_stride, void *workspace,
                                          size_t workspace_bytes, void *stream);

/* What rows of logits [rows][row_stride] (F32, BF16 or F16; rows and vocab at most 2^20,
 * rows * ceil(vocab / 2048) at most 2^26 - 4, row_stride at most 2^40) say of given tokens.
 * With p = softmax of a row:
 *   logprob  F32 [rows], ln p of tokens[r] (device uint32 [rows]); NaN where that is no
 *            token of the vocabulary
 *   rank     uint32 [rows], how many tokens come before it in the order of evo_sampler_sample
 *            (logits descending, equal ones by ascending index); UINT32_MAX where
 *            logprob is NaN
 *   entropy  F32 [rows], -sum p ln p, in nats
 *   top_tokens, top_logprobs  uint32 and F32 [rows][alternatives], the first tokens of
 *            that order and their ln p; alternatives at most 64 and vocab
 * Each output may be NULL (tokens too, if logprob and rank are; the last two only when
 * alternatives is 0), but not all. A token whose logit is -infinity has p = 0 and ln p =
 * -infinity. A row that holds NaN or +infinity, or nothing above -infinity, gets NaN and
 * UINT32_MAX throughout. Sums are F32 and leave out the largest logit's own 1, so that ln p of
 * a token that the row is sure of keeps its relative precision, down to 2^-126, below which
 * a weight counts as none.
 * The workspace (16-byte aligned, no initial contents) is needed above a vocabulary of
 * 2048; its size is 0 below, and for rows and vocabularies that are refused. Calls that
 * overlap need one each. */
EVO_API size_t evo_hip_token_logprobs_workspace_bytes(size_t rows, size_t vocab,
                                                      size_t alternatives);
EVO_API evo_status evo_hip_token_logprobs(evo_hip_dtype dtype, const void *logits, size_t rows,
                                          size_t vocab, size_t row_stride,
                                          const uint32_t *tokens, float *logprob, uint32_t *rank,
                                          float *entropy, size_t alternatives,
                                          uint32_t *top_tokens, float *top_logprobs,
                                          void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif
