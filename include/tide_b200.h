/*
 * tide_b200.h -- C ABI of the B200 (sm_100a) early-exit hot path.
 *
 * Everything here takes plain device pointers, sizes and a CUDA stream
 * handle; no framework types cross this boundary.  Every call enqueues work
 * on `stream` (NULL = legacy default stream) and returns without waiting.
 * Return value: TIDE_OK (0) or a TIDE_ERR_* code; tide_last_error() gives a
 * message for the calling thread.  Faults the kernels detect on the device
 * (an exit position outside the output buffer, a look-back wait that ran out)
 * are reported through the optional `error_word` (device int32, bit mask of
 * TIDE_DEVERR_*): the affected write is skipped, the kernel returns, and the
 * word is read back by the caller at its next synchronisation point.
 *
 * Reference interfaces replaced (RightNow-AI/TIDE v0.2.1):
 *   tide_fused_layernorm_route  <- torch.ops.tide.fused_layernorm_route
 *                                  csrc/extensions/torch_bindings.cpp:77-134,298-299
 *   tide_batch_compact          <- torch.ops.tide.batch_compact
 *                                  csrc/extensions/torch_bindings.cpp:136-198,300
 *   tide_exit_scatter           <- torch.ops.tide.exit_scatter
 *                                  csrc/extensions/torch_bindings.cpp:200-243,301-302
 *   tide_exit_projection        <- torch.ops.tide.exit_projection
 *                                  csrc/extensions/torch_bindings.cpp:245-293,303-304
 *   tide_checkpoint             <- one checkpoint of TIDERuntime.forward:
 *                                  python/TIDE/runtime.py:168-180 (score, strict
 *                                  '>' threshold, normed exit scatter) with the
 *                                  compaction of SkipScheduler.process_exits,
 *                                  python/TIDE/scheduler.py:63-102
 *   tide_norm_scatter           <- final norm + scatter of the rows that never
 *                                  exit: python/TIDE/runtime.py:183-187,
 *                                  python/TIDE/scheduler.py:111-116
 *   tide_router_fold            <- the per-call weight casts/transposes of
 *                                  torch_bindings.cpp:101-103 and the
 *                                  pre-transpose of runtime.py:85-87, done once
 */
#ifndef TIDE_B200_H
#define TIDE_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *tide_stream_t; /* a cudaStream_t */

enum tide_dtype { TIDE_DTYPE_F32 = 0, TIDE_DTYPE_F16 = 1, TIDE_DTYPE_BF16 = 2 };
enum tide_norm { TIDE_NORM_RMS = 0, TIDE_NORM_LAYER = 1 };
/* TIDE_PATH_TC: the single-pass fused cluster kernel (bf16/fp16, router width
 * 128, hidden size with a resident weight slice); TIDE_PATH_TC_SPLIT: the
 * tensor-core router followed by the stable-partition kernel; TIDE_PATH_SIMT:
 * fp32 SIMT router + partition (any dtype and shape). */
enum tide_path { TIDE_PATH_AUTO = 0, TIDE_PATH_SIMT = 1, TIDE_PATH_TC = 2, TIDE_PATH_TC_SPLIT = 3 };

enum tide_status {
  TIDE_OK = 0,
  TIDE_ERR_INVALID = 1,     /* bad argument (null pointer, size, dtype)   */
  TIDE_ERR_UNSUPPORTED = 2, /* valid but not handled by the chosen path    */
  TIDE_ERR_CUDA = 3,        /* a CUDA runtime call failed                  */
  TIDE_ERR_WORKSPACE = 4,   /* workspace missing, too small or misaligned  */
  TIDE_ERR_ALIGNMENT = 5    /* pointer/stride not 16-byte aligned          */
};

/* device-side error bits written to error_word */
enum tide_device_error {
  TIDE_DEVERR_POSITION = 1, /* exit position outside [0, n_total): row skipped */
  TIDE_DEVERR_TIMEOUT = 2,  /* a bounded spin wait expired; results invalid  */
  TIDE_DEVERR_COUNT = 4,    /* device row count above the row capacity       */
  TIDE_DEVERR_PAGES = 8     /* no free page, or a block table too narrow     */
};

int tide_abi_version(void);
const char *tide_last_error(void);

/* ---- reference operator set ------------------------------------------- */

/* scores[i] = sigmoid(up . SiLU(down_t^T . (RMSNorm(input[i]) * norm_weight)))
 * input [n_tokens, hidden_dim] of `dtype`; norm_weight [hidden_dim] fp32;
 * down_weight_t [hidden_dim, bottleneck_dim] fp32 (the pre-transposed layout
 * of runtime.py:85-87); up_weight_t [bottleneck_dim] fp32; scores [n] fp32.
 * bottleneck_dim <= 256, as in fused_layernorm_route.cu:104-168. */
int tide_fused_layernorm_route(int dtype, const void *input, const float *norm_weight,
                               const float *down_weight_t, const float *up_weight_t,
                               float eps, float *scores, int64_t n_tokens,
                               int64_t hidden_dim, int64_t bottleneck_dim,
                               tide_stream_t stream);

/* Stable split of rows by exit_mask (non-zero = exit).  Rows with mask 0 go
 * to compacted[0..num_remaining) with their source index in
 * continue_indices; rows with mask != 0 go to exited[0..n-num_remaining)
 * with their index in exit_indices.  Both orders are ascending source order.
 * compacted/exited have room for n_tokens rows.  num_remaining: device int32. */
size_t tide_batch_compact_workspace_size(int64_t n_tokens);
int tide_batch_compact(int dtype, const void *input, const int32_t *exit_mask,
                       void *compacted, void *exited, int32_t *continue_indices,
                       int32_t *exit_indices, int32_t *num_remaining, int64_t n_tokens,
                       int64_t hidden_dim, void *workspace, size_t workspace_bytes,
                       int32_t *error_word, tide_stream_t stream);

/* tide_batch_compact for callers that cannot allocate device memory: the
 * same split, outputs and argument meaning, but no workspace argument.  For
 * hosts that only lend the library the tensors they pass in (an FFI host
 * whose GPU memory belongs to another runtime, code running where allocation
 * is forbidden).  It has no counterpart in the reference.
 * Its look-back scratch is a file-scope device array sized for at most
 * TIDE_NOALLOC_MAX_ROWS rows (65,792 bytes, held by every GPU that loads the
 * library until exit); larger n_tokens is rejected with TIDE_ERR_INVALID.  It
 * calls no allocator.  The first call on a device looks the array's address
 * up (make it before any stream capture) and keeps it for the life of the
 * process: after a cudaDeviceReset (or anything else that destroys and
 * recreates the device's primary context) the kept address is stale, so do
 * not call this entry point on that device again in the same process.  All
 * calls on a device share the array: calls whose kernels overlap on the GPU
 * race, so serialise them. */
#define TIDE_NOALLOC_MAX_ROWS 1048576
int tide_batch_compact_noalloc(int dtype, const void *input, const int32_t *exit_mask,
                               void *compacted, void *exited, int32_t *continue_indices,
                               int32_t *exit_indices, int32_t *num_remaining, int64_t n_tokens,
                               int64_t hidden_dim, int32_t *error_word, tide_stream_t stream);

/* output_buffer[exit_positions[i]] = exited_states[i]  (bit copy) */
int tide_exit_scatter(int dtype, const void *exited_states, const int32_t *exit_positions,
                      void *output_buffer, int64_t n_exited, int64_t hidden_dim,
                      int64_t n_total, int32_t *error_word, tide_stream_t stream);

/* output_buffer[exit_positions[i]] = RMSNorm(exited_states[i]) * norm_weight,
 * computed in fp32 and rounded to `dtype`. */
int tide_exit_projection(int dtype, const void *exited_states, const float *norm_weight,
                         const int32_t *exit_positions, void *output_buffer, float eps,
                         int64_t n_exited, int64_t hidden_dim, int64_t n_total,
                         int32_t *error_word, tide_stream_t stream);

/* output_buffer[positions[i]] = final_norm(rows[i]) rounded to `dtype`, the
 * final norm being RMSNorm (norm_bias ignored) or LayerNorm (norm_bias may be
 * NULL), statistics in fp32.  The remaining-token step of TIDERuntime.forward,
 * python/TIDE/runtime.py:183-187, and SkipScheduler.finalize,
 * python/TIDE/scheduler.py:111-116. */
int tide_norm_scatter(int dtype, int norm_type, const void *rows, const int64_t *positions,
                      void *output_buffer, const float *norm_weight, const float *norm_bias,
                      float eps, int64_t n_rows, int64_t hidden_dim, int64_t n_total,
                      int32_t *error_word, tide_stream_t stream);

/* Rows of a full tensor picked through an index, for a live row count kept
 * on the device (checkpoint k-1's counts_out), so that checkpoints chain
 * without a host read-back.  i runs over [0, *n_rows_dev) (clamped to
 * n_rows; [0, n_rows) when n_rows_dev is NULL); an index outside [0, n_src)
 * skips the row and sets TIDE_DEVERR_POSITION.
 * tide_gather_rows:       dst[i] = src[index[i]], src [n_src, H]: the still-
 *                         active rows of a later layer's hidden states, the
 *                         `hidden[~exited]` of python/TIDE/runtime.py:172-174
 *                         (and of scheduler.py:98 in the live loop).
 * tide_norm_at_positions: out[positions[i]] = final_norm(src[positions[i]]),
 *                         src and out [n_total, H]: the rows that never exit,
 *                         python/TIDE/runtime.py:183-187. */
int tide_gather_rows(int dtype, const void *src, int64_t n_src, const int64_t *index,
                     const int32_t *n_rows_dev, int64_t n_rows, int64_t hidden_dim, void *dst,
                     int32_t *error_word, tide_stream_t stream);
int tide_norm_at_positions(int dtype, int norm_type, const void *src, const int64_t *positions,
                           const int32_t *n_rows_dev, int64_t n_rows, int64_t hidden_dim,
                           int64_t n_total, void *output_buffer, const float *norm_weight,
                           const float *norm_bias, float eps, int32_t *error_word,
                           tide_stream_t stream);

/* Decode attention over a KV cache addressed by slot: for each of the n_rows
 * rows still active in a decode step (their slot ids as compacted by
 * tide_checkpoint's slots_out),
 *   out[i, h] = softmax_j(scale * q[i, h] . K[slots[i], h/G, j]) . V[slots[i], h/G, j],
 *   j in [0, length), G = n_q_heads / n_kv_heads (at most 8), head_dim 128.
 * q, out [n_rows, n_q_heads, 128]; K, V caches [n_slots, n_kv_heads, max_len, 128],
 * bf16 or fp16.  Positions a sequence skipped hold zeros and count like any
 * other (the "zero_pad" K/V policy of python/TIDE/runtime.py:194-221).  It
 * replaces, for the rows that have not exited, the attention of the HF model
 * call inside the reference's decode loop (runtime.py:266-273).  A slot
 * outside [0, n_slots) skips its row and sets TIDE_DEVERR_POSITION.
 * n_rows_dev (optional, device int32): only rows below it are computed (the
 * live count a checkpoint wrote).  length_dev (optional, device int32): the
 * length is read from the device, clamped to [1, length]; `length` then only
 * bounds it (shared memory is sized for it).  Both keep a decode step free of
 * host values, so it can be captured in a CUDA graph. */
int tide_decode_attention(int dtype, const void *q, const void *k_cache, const void *v_cache,
                          const int32_t *slots, void *out, int64_t n_rows,
                          const int32_t *n_rows_dev, int64_t n_q_heads, int64_t n_kv_heads,
                          int64_t head_dim, int64_t n_slots, int64_t max_len, int64_t length,
                          const int32_t *length_dev, float scale, int32_t *error_word,
                          tide_stream_t stream);

/* Append one decode position to a KV cache addressed by slot:
 *   K[slots[i], h, pos, :] = k_new[i, h, :],  V[...] = v_new[i, h, :]
 * for i below the live row count (*n_rows_dev clamped to [0, n_rows]; n_rows
 * when NULL) and pos = *position_dev when given, else `position`.  k_new,
 * v_new [n_rows, n_kv_heads, 128]; caches as tide_decode_attention's.  A
 * position outside [0, max_len) or a slot outside [0, n_slots) writes
 * nothing for the rows concerned and sets TIDE_DEVERR_POSITION.  With the
 * checkpoint's compacted slot ids it stores the keys and values of the rows
 * still active in a decode step; an exited row's entry at that position
 * keeps the zeros it was created with (the reference's "zero_pad",
 * python/TIDE/runtime.py:194-221). */
int tide_kv_append(int dtype, const void *k_new, const void *v_new, const int32_t *slots,
                   const int32_t *n_rows_dev, int64_t n_rows, int64_t n_kv_heads,
                   int64_t head_dim, void *k_cache, void *v_cache, int64_t n_slots,
                   int64_t max_len, int64_t position, const int32_t *position_dev,
                   int32_t *error_word, tide_stream_t stream);

/* tide_norm_scatter with the row count on the device:
 *   output_buffer[positions[i]] = final_norm(rows[i]),  i < *n_rows_dev
 * (clamped to [0, n_rows]; n_rows when NULL).  The finalize step
 * (python/TIDE/scheduler.py:102-120) for survivors whose count a checkpoint
 * left on the device.  A position outside [0, n_total) skips its row and
 * sets TIDE_DEVERR_POSITION. */
int tide_norm_scatter_rows(int dtype, int norm_type, const void *rows, const int64_t *positions,
                           const int32_t *n_rows_dev, int64_t n_rows, int64_t hidden_dim,
                           int64_t n_total, void *output_buffer, const float *norm_weight,
                           const float *norm_bias, float eps, int32_t *error_word,
                           tide_stream_t stream);

/* The elementwise work of a Llama-family decode layer for the live decoder,
 * each rounding where the HF module it replaces rounds (bf16 or fp16 rows,
 * weights in the rows' type), rows below the live count only (*n_rows_dev
 * clamped to [0, n_rows]; n_rows when NULL):
 * tide_rms_norm:      s = x, or s = to_T(x + delta) written to sum_out (when
 *                     given); out = to_T(w * to_T(s * rsqrt(mean(s^2) + eps)))
 *                     -- HF LlamaRMSNorm / Qwen3RMSNorm with an optional fused
 *                     residual add.  hidden_dim % 8 == 0, <= 8192.
 * tide_qk_norm_rope:  q [n, hq, 128], k, v [n, hkv, 128], rows q_row_stride
 *                     and kv_row_stride elements apart (0: packed; k and v
 *                     share a stride, so q, k and v may be column slices of
 *                     one fused projection's output): optional per-head
 *                     RMSNorm of q and k (Qwen3 q_norm / k_norm; NULL weight =
 *                     none), the rotary embedding q*cos + rotate_half(q)*sin
 *                     with cos/sin = to_T(cos/sin(pos * inv_freq[j]) *
 *                     attention_scaling), then q to q_out and k, v into the
 *                     slot-addressed caches at pos (*position_dev when given).
 *                     rope_positions (optional, int64 per row): each row's own
 *                     rotary position instead of pos, and q written to
 *                     q_out[slots[i]] instead of q_out[i] (a prefill, which
 *                     passes [tokens, heads, 1, 128] buffers as the caches,
 *                     its rows' token indices as the slots and pos 0, so
 *                     that q, k and v land at their tokens' places).  A slot
 *                     or position outside the cache writes nothing for that
 *                     row and sets TIDE_DEVERR_POSITION.
 * tide_silu_mul:      out = to_T(to_T(silu(gate)) * up), [n, width], width % 8
 *                     == 0 -- the gated MLP's act_fn(gate_proj(x)) * up_proj(x).
 * The reference runs the model's own modules for these inside its decode
 * loop (python/TIDE/runtime.py:266-273). */
int tide_rms_norm(int dtype, const void *x, const void *delta, void *sum_out, const void *weight,
                  void *out, int64_t n_rows, const int32_t *n_rows_dev, int64_t hidden_dim,
                  float eps, tide_stream_t stream);
int tide_qk_norm_rope(int dtype, const void *q, const void *k, const void *v,
                      int64_t q_row_stride, int64_t kv_row_stride,
                      const void *q_norm_weight, const void *k_norm_weight, float eps,
                      const float *inv_freq, float attention_scaling, int64_t position,
                      const int32_t *position_dev, const int64_t *rope_positions,
                      const int32_t *slots, const int32_t *n_rows_dev, int64_t n_rows,
                      int64_t n_q_heads,
                      int64_t n_kv_heads, int64_t head_dim, void *q_out, void *k_cache,
                      void *v_cache, int64_t n_slots, int64_t max_len, int32_t *error_word,
                      tide_stream_t stream);
int tide_silu_mul(int dtype, const void *gate, const void *up, void *out, int64_t n_rows,
                  const int32_t *n_rows_dev, int64_t width, tide_stream_t stream);

/* ---- ragged batches over a paged cache ---------------------------------- */
/*
 * Sequences of different lengths, packed: sequence i holds the token rows
 * [cu_seqlens[i], cu_seqlens[i + 1]) (device int32, n_seqs + 1 entries,
 * ascending).  Rows behind the last sequence are left as they were.
 *
 * A paged cache keeps a request's keys (and, in a second array, its values)
 * in pages [n_pages, n_kv_heads, page_size, head_dim] of the rows' type:
 * position p of request r lies in page block_tables[r * max_pages +
 * p / page_size], at p % page_size.  A page with one KV head is one
 * contiguous run, as a slot of the caches of tide_decode_attention is.  A
 * page holds one request's positions; the entries of a block table past a
 * request's last page are not read, nor is what lies in its last page past
 * its length.  The reference has no such cache: its decode loop keeps the
 * model's own (python/TIDE/runtime.py:223-313) and takes one length for the
 * whole batch.
 *
 * tide_packed_attention: causal attention within each packed sequence,
 *   out[i, h] = (sum_j e^(s_ij) v[j, h / G]) / (zero_keys[i] + sum_j e^(s_ij)),
 *   s_ij = scale * q[i, h] . k[j, h / G],  j over the rows of i's sequence up
 *   to i,  G = n_q_heads / n_kv_heads (any whole number).
 * zero_keys (optional, int32 per row; negative counts as 0): so many further
 * keys that are zero, as are their values.  With the survivors of a
 * checkpoint as the rows and, for each, its position minus its rank among
 * its sequence's survivors, this is attention over the whole sequence whose
 * exited tokens are zero-padded (python/TIDE/runtime.py:194-221), without
 * the zeros.
 *
 * tide_paged_attention: the new tokens of each request over its paged cache,
 * which already holds their own keys and values:
 *   new token t of sequence i (of n_i rows) sees the positions [0, L - n_i +
 *   t], L = kv_lens[r], r = seq_ids[i] (i when NULL); a token that sees none
 *   gets zeros.
 * cu_seqlens NULL: one row per sequence (a decode step).  n_seqs_dev
 * (optional): only the sequences below it run.  max_kv_len bounds the
 * lengths, and sizes the workspace and the split of long contexts; a longer
 * one counts as invalid.
 *
 * Both: bf16 or fp16, head_dim 64 or 128, scale > 0, up to 128 query heads
 * per KV head; page_size a power of two of at least 16.  q, k, v: heads
 * packed within a row, rows q_row_stride and kv_row_stride elements apart
 * (0: packed; multiples of 8, so that column slices of one projection's
 * output do).  A sequence with bad bounds, a request outside
 * [0, n_requests), or a length outside [0, max_kv_len] is skipped, its rows
 * left as they were, and sets TIDE_DEVERR_POSITION; a page outside
 * [0, n_pages) reads as zeros and sets it too.  A NaN or infinity in a value
 * row reaches the tokens that see that row, and no others (the weights are
 * rounded to the rows' type: an infinity whose weight rounds to 0, 2^-32 of the
 * largest or less in fp16, arrives as a NaN). */
int tide_packed_attention(int dtype, const void *q, const void *k, const void *v,
                          int64_t q_row_stride, int64_t kv_row_stride, const int32_t *cu_seqlens,
                          int64_t n_seqs, const int32_t *zero_keys, void *out, int64_t n_tokens,
                          int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, float scale,
                          int32_t *error_word, tide_stream_t stream);
size_t tide_paged_attention_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t n_q_heads,
                                           int64_t n_kv_heads, int64_t head_dim,
                                           int64_t max_kv_len);
int tide_paged_attention(int dtype, const void *q, int64_t q_row_stride, const void *k_cache,
                         const void *v_cache, int64_t n_pages, int64_t page_size,
                         const int32_t *block_tables, int64_t max_pages, int64_t n_requests,
                         const int32_t *kv_lens, const int32_t *cu_seqlens, const int32_t *seq_ids,
                         int64_t n_seqs, const int32_t *n_seqs_dev, void *out, int64_t n_tokens,
                         int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                         int64_t max_kv_len, float scale, void *workspace, size_t workspace_bytes,
                         int32_t *error_word, tide_stream_t stream);

/* Keys and values of new tokens into a paged cache: row i of k_new and v_new
 * [n_rows, n_kv_heads, head_dim] (rows kv_row_stride elements apart; 0:
 * packed) goes to slot s = slot_map[row_ids[i]] (slot_map[i] when row_ids is
 * NULL), that is to page s / page_size at s % page_size, for i below
 * *n_rows_dev (clamped to [0, n_rows]; n_rows when NULL).  k_new and v_new
 * both NULL write zeros (the keys and values of exited tokens,
 * python/TIDE/runtime.py:194-221).  A slot of -1 is skipped; any other slot
 * outside the cache, or a row id outside [0, n_slot_map), skips its row and
 * sets TIDE_DEVERR_POSITION.  No slot may be named twice in a call.  head_dim
 * 64 or 128, bf16 or fp16, any page size; 16-byte aligned rows. */
int tide_paged_append(int dtype, const void *k_new, const void *v_new, int64_t kv_row_stride,
                      const int64_t *slot_map, int64_t n_slot_map, const int32_t *row_ids,
                      const int32_t *n_rows_dev, int64_t n_rows, int64_t n_kv_heads,
                      int64_t head_dim, void *k_cache, void *v_cache, int64_t n_pages,
                      int64_t page_size, int32_t *error_word, tide_stream_t stream);

/* ---- a paged cache in 4 bits -------------------------------------------- */
/*
 * The same pages with keys and values in 4.5 bits each, for bf16 and fp16 rows.
 * A group is 32 neighbouring channels of a token's key or value in one head;
 * it has codes c and a zero point z in 0..15 and a scale s, and stands for
 * (c - z) s, which both 16-bit types hold exactly.  With lo and hi the group's
 * least and largest value, 0 among them, and t = (hi - lo) / 15:
 *   s = t rounded up to four significant bits (0 for a group of zeros, else at
 *   least 2^-120, 2^-21 for fp16 rows),  z = round(-lo / s),
 *   c = min(max(round(x / s) + z, 0), 15)    (ties to even).
 * So a value is off by s / 2 at most (by s where s / 2 more would pass the rows'
 * largest number), and zero is held as zero.  A group with a value that is not
 * finite in the rows' type reads as NaN (a key after its norm and rotation).  A
 * cache is read as the type that it was written from.
 *
 * The cache is [n_pages, n_kv_heads, page_size / 16, 18 head_dim] bytes.  The 18
 * head_dim bytes of 16 tokens of a head: the codes of the keys
 * [16, head_dim / 2], of the values, the scales of the keys [head_dim / 32,
 * token % 4, token / 4] of 16 bits, of the values.  Eight channels are 32 bits
 * (little-endian), four each, lowest first channels 0, 2, 4, 6, 1, 3, 5, 7.  A
 * scale is a bf16 with z in its last four bits.  All bytes zero is a cache of
 * zeros.
 *
 * tide_paged_append_q4: keys and values of new tokens into it, as
 * tide_paged_append, with what comes before on the way.  Row i is entry m =
 * row_ids[i] (i when NULL) of slot_map and positions.  k_new row i, with its
 * heads' RMSNorm (k_norm_weight [head_dim] of the rows' type, or NULL: none)
 * and turned by its position (inv_freq [head_dim / 2] fp32, or NULL: not),
 *   y = x * rsqrt(mean(x^2) + eps) * w,
 *   out[j] = y[j] cos a - y[j + d/2] sin a,  out[j + d/2] = y[j + d/2] cos a +
 *   y[j] sin a,  a = positions[m] * inv_freq[j],  cos and sin times
 *   attention_scaling,
 * goes to slot slot_map[m] with v_new row i as it is.  q row i (optional, with
 * q_norm_weight) is treated likewise and goes to row i of q_out [n_rows,
 * n_q_heads, head_dim], whatever its slot; rows not below *n_rows_dev, and
 * those of a row id outside [0, n_slot_map), are left.  Nothing is rounded on
 * the way: q once to its type, k once to 32 bits before its codes are made, the
 * angle being taken in 64 bits.  q, k_new and v_new all NULL write zeros.
 * Slots and row ids as in tide_paged_append; no slot may be named twice in a
 * call.  page_size a multiple of 16.
 *
 * tide_paged_read_q4: the key and value at slots[i] to row i of k_out and v_out
 * [n_rows, n_kv_heads, head_dim]; a row with slot -1 is left as it was, one
 * with a slot outside the cache too (TIDE_DEVERR_POSITION).
 *
 * tide_paged_attention_q4: tide_paged_attention over it, with the same
 * arguments and rules.  A key or value group that reads as NaN reaches the tokens
 * that see it, and no others.  Where sequences may have many rows the workspace
 * holds contexts in 16 bits: up to 256 MB, or those of one sequence of max_kv_len
 * keys if they are more. */
int tide_paged_append_q4(int dtype, const void *q, int64_t q_row_stride, const void *k_new,
                         const void *v_new, int64_t kv_row_stride, const void *q_norm_weight,
                         const void *k_norm_weight, float eps, const float *inv_freq,
                         float attention_scaling, const int64_t *positions,
                         const int64_t *slot_map, int64_t n_slot_map, const int32_t *row_ids,
                         const int32_t *n_rows_dev, int64_t n_rows, int64_t n_q_heads,
                         int64_t n_kv_heads, int64_t head_dim, void *q_out, void *cache,
                         int64_t n_pages, int64_t page_size, int32_t *error_word,
                         tide_stream_t stream);
int tide_paged_read_q4(int dtype, const void *cache, int64_t n_pages, int64_t page_size,
                       const int64_t *slots, int64_t n_rows, int64_t n_kv_heads, int64_t head_dim,
                       void *k_out, void *v_out, int32_t *error_word, tide_stream_t stream);
size_t tide_paged_attention_q4_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t n_requests,
                                              int64_t n_q_heads, int64_t n_kv_heads,
                                              int64_t head_dim, int64_t max_kv_len);
int tide_paged_attention_q4(int dtype, const void *q, int64_t q_row_stride, const void *cache,
                            int64_t n_pages, int64_t page_size, const int32_t *block_tables,
                            int64_t max_pages, int64_t n_requests, const int32_t *kv_lens,
                            const int32_t *cu_seqlens, const int32_t *seq_ids, int64_t n_seqs,
                            const int32_t *n_seqs_dev, void *out, int64_t n_tokens,
                            int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                            int64_t max_kv_len, float scale, void *workspace,
                            size_t workspace_bytes, int32_t *error_word, tide_stream_t stream);

/* ---- page bookkeeping --------------------------------------------------- */

/* The page bookkeeping of one step, from the requests' lengths:
 *   1. a request with done[r] != 0 (optional) gives back the pages of its
 *      context_lens[r] positions and starts over from length 0;
 *   2. every request gets the pages that new_lens[r] more positions need,
 *      written behind its present ones in block_tables [n_requests,
 *      max_pages];
 *   3. kv_lens[r] = its length with them; cu_seqlens [n_requests + 1]: the
 *      packed offsets of the new tokens; and per new token, in packed order,
 *      slot_map (its slot in the cache, page * page_size + offset) and
 *      positions (its position in its request).  Entries past the last token
 *      up to n_slots: slot -1, position 0.
 * free_pages [n_pages] is a stack whose first *n_free entries are free pages:
 * returned pages are pushed in order of request and position, new ones popped
 * in order of request and position.  The new count goes to *n_free_out.
 * kv_lens may be context_lens and n_free_out may be n_free (in place, as a
 * captured step needs it).
 * A request that needs more pages than are left, in order of requests, or
 * more than max_pages, gets none: its kv_lens entry is its old length, its
 * tokens' slots are -1, and TIDE_DEVERR_PAGES is set; once one did not find
 * its pages, no later one gets new ones.  A negative length, or a new length
 * above n_slots, counts as 0 and sets TIDE_DEVERR_COUNT, as does a free count
 * outside [0, n_pages] (clamped) and a request whose tokens end past n_slots
 * (it gets no pages).  A page returned to a full stack is dropped and sets
 * TIDE_DEVERR_PAGES.  n_requests <= 8192. */
int tide_page_tables(const int32_t *context_lens, const int32_t *new_lens, const int32_t *done,
                     int64_t n_requests, int32_t *free_pages, const int32_t *n_free,
                     int64_t n_pages, int32_t *block_tables, int64_t max_pages, int64_t page_size,
                     int32_t *n_free_out, int32_t *kv_lens, int32_t *cu_seqlens, int64_t *slot_map,
                     int64_t *positions, int64_t n_slots, int32_t *error_word,
                     tide_stream_t stream);

/* ---- router preparation (once per router) ------------------------------ */

/* From the router's down.weight [B, H] fp32 and the final norm's weight (and
 * bias, LayerNorm only) [H] fp32, build:
 *   down_t      [H, B] fp32             (SIMT path; may be NULL)
 *   folded      [B, H] in fold_dtype    folded[b,i] = down[b,i] * norm_weight[i]
 *                                       (tensor-core path; may be NULL)
 *   colsum      [B] fp32                sum_i float(folded[b,i])   (may be NULL)
 *   bias_proj   [B] fp32                sum_i norm_bias[i]*down[b,i] (may be NULL) */
int tide_router_fold(int fold_dtype, const float *down, const float *norm_weight,
                     const float *norm_bias, int64_t hidden_dim, int64_t bottleneck_dim,
                     float *down_t, void *folded, float *colsum, float *bias_proj,
                     tide_stream_t stream);

/* ---- one checkpoint of the early-exit path ----------------------------- */

typedef struct tide_checkpoint_args {
  int32_t dtype;          /* element type of x, out_buffer, compact_out        */
  int32_t norm_type;      /* TIDE_NORM_RMS or TIDE_NORM_LAYER                  */
  int32_t path;           /* TIDE_PATH_AUTO / _SIMT / _TC                        */
  int32_t reserved0;
  int64_t n_rows;         /* rows of x (capacity when n_rows_dev != NULL)      */
  int64_t hidden_dim;     /* H                                                   */
  int64_t bottleneck_dim; /* B (router width)                                    */
  int64_t n_total;        /* rows of out_buffer                                  */
  const void *x;          /* [n_rows, H] hidden states of the active tokens     */
  const int32_t *n_rows_dev; /* optional device count of valid rows (<= n_rows) */
  /* final norm */
  const float *norm_weight; /* [H] fp32                                          */
  const float *norm_bias;   /* [H] fp32, LayerNorm only, may be NULL             */
  float eps;
  /* router (from tide_router_fold) */
  float up_bias;          /* scalar added before the sigmoid (0 = reference)   */
  const float *down_t;    /* [H, B] fp32: SIMT path                            */
  const void *folded;     /* [B, H] dtype: tensor-core path                    */
  const float *colsum;    /* [B]: LayerNorm on the tensor-core path            */
  const float *bias_proj; /* [B]: LayerNorm with bias                          */
  const float *up;        /* [B] fp32 up.weight                                */
  float threshold;        /* exit iff score > threshold (strict)               */
  int32_t reserved1;
  /* token bookkeeping */
  const int64_t *positions_in; /* [n_rows] original token position; NULL = row index */
  const int32_t *slots_in;     /* [n_rows] KV slot id; may be NULL                  */
  /* outputs (each may be NULL except counts_out) */
  void *out_buffer;            /* [n_total, H]: exiting rows, final-normed       */
  void *compact_out;           /* [n_rows, H]: surviving rows, stable order      */
  int64_t *positions_out;      /* [n_rows]: surviving rows' positions            */
  int32_t *slots_out;          /* [n_rows]: surviving rows' slots                */
  int64_t *exit_positions_out; /* [n_rows]: exiting rows' positions, stable      */
  float *scores_out;           /* [n_rows]: router scores                        */
  int32_t *counts_out;         /* [2] device: {survivors, exits}                 */
  int32_t *error_word;         /* device int32 bit mask, may be NULL             */
  void *workspace;             /* from tide_checkpoint_workspace_size            */
  size_t workspace_bytes;
} tide_checkpoint_args;

size_t tide_checkpoint_workspace_size(const tide_checkpoint_args *args);
int tide_checkpoint(const tide_checkpoint_args *args, tide_stream_t stream);

/* Which path tide_checkpoint would take for these arguments (TIDE_PATH_SIMT,
 * TIDE_PATH_TC or TIDE_PATH_TC_SPLIT), or a negative TIDE_ERR_* code. */
int tide_checkpoint_select_path(const tide_checkpoint_args *args);

#ifdef __cplusplus
}
#endif

#endif /* TIDE_B200_H */
