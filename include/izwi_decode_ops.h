/*
 * izwi_decode_ops — the decode-step neighbours of the quantized projections: RMSNorm, the
 * q/k head norm, rotary embedding and single-token grouped-query attention, f32 and f16; for several
 * continuations of one prompt a quantized key / value cache, the attention over it and beam search's selection.
 *
 * Each entry point is the device side of one of the reference's fused-kernel hooks
 * (crates/izwi-core/src/kernels/mod.rs:109-225), which today dispatch to Metal only
 * (crates/izwi-core/src/kernels/metal.rs) and return None elsewhere, so that the caller falls
 * back to Candle's eager operators.  Arithmetic follows the reference's shaders
 * (metal.rs:59-381) in f32; only the order of the sums differs (the reference's tests allow
 * 1e-5 against the eager operators, metal.rs:2956).
 *
 * Conventions are those of izwi_qmm.h: return IZWI_QMM_OK or a negative izwi_qmm_status, message
 * through izwi_qmm_last_error(); `mem_space` says whether the pointers are device or host
 * memory (host buffers are staged, synchronous); `stream` is a hipStream_t or NULL.  All tensors
 * are contiguous row-major, f32 unless the entry point's name says f16.  Outputs may alias the corresponding inputs (in-place).
 */
#ifndef IZWI_DECODE_OPS_H
#define IZWI_DECODE_OPS_H

#include <stdint.h>

#include "izwi_qmm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* `try_fused_rms_norm(input, weight, eps)` (kernels/mod.rs:141-155, metal.rs:1979-2024, shader
 * metal.rs:147-186): y[r, i] = x[r, i] * rsqrt(mean_i(x[r, :]^2) + eps) * weight[i] for `rows` rows
 * of `hidden` values.  The reference refuses rows == 0 and hidden == 0 (returns None): here rows ==
 * 0 is a no-op and hidden == 0 is IZWI_QMM_ERR_INVALID. */
int izwi_rms_norm_f32(const float* x, const float* weight, int64_t rows, int64_t hidden, float eps,
                      float* y, int mem_space, void* stream);

/* `try_fused_qk_rms_norm(q, k, qk_weight, eps)` (kernels/mod.rs:109-123, metal.rs:1906-1975,
 * shader metal.rs:59-101): the per-head norms of Qwen3 attention (qwen3/core.rs:1470) in one
 * launch.  q is `[q_rows, head_dim]` (q_rows = batch * heads for one token), k is
 * `[k_rows, head_dim]`, qk_weight is `[2 * head_dim]`: q's weights, then k's.  The reference's
 * shader is limited to head_dim <= 256 and one token; this kernel takes any row counts and
 * head_dim <= 8192. */
int izwi_qk_rms_norm_f32(const float* q, const float* k, const float* qk_weight, int64_t q_rows,
                         int64_t k_rows, int64_t head_dim, float eps, float* q_out, float* k_out,
                         int mem_space, void* stream);

/* `try_fused_rope_pair_bshd(q, k, cos_sin)` (kernels/mod.rs:157-171, metal.rs:2026-2094, shader
 * metal.rs:227-265): q is `[batch, seq, q_heads, head_dim]`, k is `[batch, seq, k_heads,
 * head_dim]`, cos_sin is `[seq, head_dim]` with the cosines in the first half of a row and the
 * sines in the second; head_dim even.  The two halves of a head rotate against each other:
 * out[d] = x[d] cos[d] - x[half + d] sin[d], out[half + d] = x[d] sin[d] + x[half + d] cos[d]. */
int izwi_rope_pair_bshd_f32(const float* q, const float* k, const float* cos_sin, int64_t batch,
                            int64_t seq, int64_t q_heads, int64_t k_heads, int64_t head_dim,
                            float* q_out, float* k_out, int mem_space, void* stream);

/* The hooks' `DType::F16` arm (the reference's `*_f16` shaders, metal.rs:103-144, 187-225, 267-305,
 * 383-457): the same four operations on IEEE half tensors (raw bits as uint16_t), every tensor of a
 * call f16 as the reference's wrappers require; values are widened on load, all arithmetic is f32
 * and each result is rounded to f16 once.  The reference's tests allow 5e-3 for this arm
 * (metal.rs:2956).  Shapes, limits and error behaviour are those of the f32 entry points. */
int izwi_rms_norm_f16(const uint16_t* x, const uint16_t* weight, int64_t rows, int64_t hidden, float eps,
                      uint16_t* y, int mem_space, void* stream);

/* izwi_rms_norm_f32 whose result goes, quantized, straight into the activation records of the batched
 * decode kernels (izwi_qmm.h, "activation records"): the layer norm in front of q|k|v and gate|up
 * (qwen3/core.rs:1866, 1877) and the quantization inside the following `QMatMul::forward` as one
 * launch.  The records equal izwi_qmm_quantize_records_f32(izwi_rms_norm_f32(x)) bit for bit.  f32,
 * device pointers, hidden a multiple of 256 up to 16384, 16-byte aligned buffers. */
int izwi_rms_norm_quantize_records_f32(int ggml_weight_dtype, const float* x, const float* weight, int64_t rows,
                                       int64_t hidden, float eps, void* records, void* stream);
int izwi_qk_rms_norm_f16(const uint16_t* q, const uint16_t* k, const uint16_t* qk_weight, int64_t q_rows,
                         int64_t k_rows, int64_t head_dim, float eps, uint16_t* q_out, uint16_t* k_out,
                         int mem_space, void* stream);
int izwi_rope_pair_bshd_f16(const uint16_t* q, const uint16_t* k, const uint16_t* cos_sin, int64_t batch,
                            int64_t seq, int64_t q_heads, int64_t k_heads, int64_t head_dim,
                            uint16_t* q_out, uint16_t* k_out, int mem_space, void* stream);
int izwi_decode_gqa_attention_f16(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t num_heads,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t kv_len,
                                  int64_t kv_capacity, float scale, uint16_t* out, int mem_space,
                                  void* stream);

/* The single-token sequence of `Qwen3Attention::forward` between the q/k/v projections and the
 * attention itself as ONE launch: `apply_qk_norm_pair` (qwen3/core.rs:1464-1478), `apply_rope_pair`
 * (core.rs:1480-1575) and the append of the new key / value rows to the cache.  q is `[num_heads,
 * head_dim]`, k and v are `[num_kv_heads, head_dim]` (the projections' outputs), qk_weight is
 * `[2 * head_dim]` (q's norm weights, then k's), cos_sin is `[head_dim]` for this position
 * (cos | sin).  Writes the normed, rotated q to q_out (may be q), the normed, rotated k and the
 * unchanged v to position `pos` of the head-major caches `[num_kv_heads, kv_capacity, head_dim]`.
 * Values are those of izwi_qk_rms_norm_f32 followed by izwi_rope_pair_bshd_f32 up to the order
 * of the norm's sum.  Device pointers only (the caches live on the device).  It has no single counterpart among the
 * reference's hooks: it is their composition for one token. */
int izwi_qk_norm_rope_append_f32(const float* q, const float* k, const float* v, const float* qk_weight,
                                 const float* cos_sin, int64_t num_heads, int64_t num_kv_heads,
                                 int64_t head_dim, float eps, float* q_out, float* k_cache, float* v_cache,
                                 int64_t kv_capacity, int64_t pos, void* stream);

/* The same sequence AND the attention behind it as one launch (two when the positions are split):
 * the attention kernel norms and rotates its query heads and the new key itself, takes the new
 * (key, value) as position `pos` and appends them to the caches on its way.  Arguments as
 * izwi_qk_norm_rope_append_f32 (without q_out) and izwi_decode_gqa_attention_f32 with
 * kv_len = pos + 1; out is `[num_heads, head_dim]`.  Results are those of the two calls bit for bit
 * (the same arithmetic in the same order) where out shares no memory with the inputs.  Device pointers only; head_dim 64, 128 or 256. */
int izwi_decode_attention_step_f32(const float* q, const float* k, const float* v, const float* qk_weight,
                                   const float* cos_sin, int64_t num_heads, int64_t num_kv_heads,
                                   int64_t head_dim, float eps, float* k_cache, float* v_cache,
                                   int64_t kv_capacity, int64_t pos, float scale, float* out, void* stream);

/* `try_fused_decode_gqa_attention_with_kv_len(q, k, v, num_heads, num_kv_heads, head_dim, kv_len,
 * scale)` (kernels/mod.rs:199-225, metal.rs:2121-2193, shader metal.rs:307-381): attention of one
 * query token.  q is `[1, num_heads, 1, head_dim]`, k and v are `[1, num_kv_heads, kv_capacity,
 * head_dim]` (head-major cache) of which the first kv_len positions count; head h reads kv head
 * h / (num_heads / num_kv_heads); out is `[1, num_heads, 1, head_dim]`,
 * softmax_p((q . k_p) * scale) . v.  The reference's shader refuses kv_len > 2048; here the
 * positions are split over workgroups and merged (any kv_len).  head_dim must be 64, 128 or 256
 * (IZWI_QMM_ERR_UNSUPPORTED otherwise).  Uses the library's per-stream scratch when the positions
 * are split.  With out == q a short cache takes another form of the kernel, whose f32 sums are in another order. */
int izwi_decode_gqa_attention_f32(const float* q, const float* k, const float* v, int64_t num_heads,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t kv_len,
                                  int64_t kv_capacity, float scale, float* out, int mem_space,
                                  void* stream);

/* Greedy next token: `argmax(&logits)` after the LM head (qwen3/chat.rs:574-597,
 * qwen3/asr/mod.rs:2762-2789, i.e. `logits.argmax(D::Minus1)` as u32), on the device, so that four
 * bytes per row come back instead of the logits.  logits is `[rows, n]`, out `[rows]`: the first
 * index of the row's maximum (ties go to the smaller index, as a left-to-right scan keeps the
 * first; a NaN is never the maximum; a row of NaNs gives 0). */
int izwi_argmax_f32(const float* logits, int64_t rows, int64_t n, uint32_t* out, int mem_space, void* stream);

/* ---- several continuations of one prompt -----------------------------------------------------------------------
 *
 * Sequences that decode together from a quantized cache: `prompts` prompts of `beams` sequences each (sequence b
 * belongs to prompt b / beams; one beam per prompt is ordinary batched decoding, one prompt a batch behind a common
 * system prompt).  What the sequences of a prompt share stands once, in a cache with a slot per prompt; what each of
 * them adds stands in a cache with a slot per sequence.  Lengths are device arrays, so that a captured step can be
 * replayed while they grow.  Device pointers only throughout. */

/* Cache formats, by their ggml ids: blocks of 32 values along a head's row, an f16 scale and 8 or 4 bits a value.
 * Blocks of equal bits to the GGUF formats' (izwi_qmm_quantize_weights_f32 makes the same Q8_0 ones); a block that
 * holds an infinity or NaN, or whose scale has no f16, reads as NaN, one whose scale is zero as zeros. */
enum { IZWI_KV_Q4_0 = 2, IZWI_KV_Q8_0 = 8 };

/* Bytes of a cache of `slots` slots, each of kv_capacity positions (rounded up to 32) of num_kv_heads key and value
 * rows; head_dim 64, 128 or 256.  0 for a shape that cannot be (the message says why).  The layout is the library's
 * own; the buffer needs no clearing. */
uint64_t izwi_decode_kv_cache_bytes(int type, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity, int64_t head_dim);

/* Quantizes the rows of `batch` sequences of up to `tokens` tokens into slots first_slot, first_slot + 1, ..: row
 * (b, t) of k and v holds num_kv_heads heads of head_dim values, k_stride (v_stride) elements behind row (b, t) - 1,
 * and goes to position starts[b] + t, for t < counts[b] (counts NULL: all).  Rows outside the capacity are left out;
 * positions that no row goes to stay as they were. */
int izwi_decode_kv_append_f32(int type, const float* k, const float* v, int64_t k_stride, int64_t v_stride,
                              const int32_t* starts, const int32_t* counts, int64_t batch, int64_t tokens,
                              int64_t first_slot, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity,
                              int64_t head_dim, void* cache, void* stream);
int izwi_decode_kv_append_f16(int type, const uint16_t* k, const uint16_t* v, int64_t k_stride, int64_t v_stride,
                              const int32_t* starts, const int32_t* counts, int64_t batch, int64_t tokens,
                              int64_t first_slot, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity,
                              int64_t head_dim, void* cache, void* stream);

/* The values that positions starts[b] .. starts[b] + tokens - 1 of those slots stand for, into contiguous k and v
 * `[batch, tokens, num_kv_heads, head_dim]`; zeros from counts[b] tokens on and outside the capacity.  With `lineage`
 * (below) position p of slot s is read from the slot of beam lineage[s][p] of the same prompt (`beams` slots a prompt, at
 * most 255; zeros where there is no such beam): a beam's history in one piece. */
int izwi_decode_kv_read_f32(int type, const void* cache, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity,
                            int64_t head_dim, const uint8_t* lineage, int64_t beams, const int32_t* starts,
                            const int32_t* counts, int64_t batch, int64_t tokens, int64_t first_slot, float* k, float* v,
                            void* stream);
int izwi_decode_kv_read_f16(int type, const void* cache, int64_t slots, int64_t num_kv_heads, int64_t kv_capacity,
                            int64_t head_dim, const uint8_t* lineage, int64_t beams, const int32_t* starts,
                            const int32_t* counts, int64_t batch, int64_t tokens, int64_t first_slot, uint16_t* k,
                            uint16_t* v, void* stream);

/* Attention of one new token per sequence: softmax((q . k) * scale) . v over positions 0 .. prefix_lens[b / beams] - 1
 * of the prompt's slot of `prefix` and positions 0 .. lens[b] - 1 of slot b of `cache`, both of format `type`; either may be
 * NULL.  q is `[batch, num_heads, head_dim]`, q_stride elements from one sequence to the next; head h reads kv head
 * h / (num_heads / num_kv_heads); out is contiguous `[batch, num_heads, head_dim]` and may share no memory with the rest.  A
 * sequence without any position gives zeros, one that reads a NaN (in q, a key, a value; an infinity in q) NaN: the whole
 * head, or a value's block of 32.  Lengths above max_prefix_len (max_len), the caller's bounds, count as
 * those, negative ones as zero; the work is shared out by the bounds.  With `lineage`, `[slots][kv_capacity rounded up to
 * 32]`, position p of sequence b is in the slot of beam lineage[b][p] of its prompt; a position whose entry is no beam
 * (>= beams) does not count.  What a sequence writes before the first selection is its own: rows begin as b % beams (zeros would
 * read the first beam's positions).  The products run on the matrix cores with f32 sums; f32 queries and the weights go as
 * two f16 numbers each, 22 bits down to 2^-16 of the row's largest number in q and 2^-14 of its largest weight, fewer of
 * what is smaller; a value counts to 2^-24 of the largest of its block of 32 among 32 neighbouring positions; f16
 * results are rounded once.  Uses the library's per-stream scratch. */
int izwi_decode_shared_attention_f32(int type, const float* q, int64_t q_stride, int64_t batch, int64_t beams,
                                     int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const void* prefix,
                                     int64_t prefix_slots, int64_t prefix_capacity, const int32_t* prefix_lens,
                                     int64_t max_prefix_len, const void* cache, int64_t slots, int64_t kv_capacity,
                                     const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale,
                                     float* out, void* stream);
int izwi_decode_shared_attention_f16(int type, const uint16_t* q, int64_t q_stride, int64_t batch, int64_t beams,
                                     int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, const void* prefix,
                                     int64_t prefix_slots, int64_t prefix_capacity, const int32_t* prefix_lens,
                                     int64_t max_prefix_len, const void* cache, int64_t slots, int64_t kv_capacity,
                                     const int32_t* lens, int64_t max_len, const uint8_t* lineage, float scale,
                                     uint16_t* out, void* stream);

/* One step of beam search.  logits is `[prompts, beams, vocab]`, scores the beams' sums of log-probabilities so far
 * `[prompts, beams]`; candidate (w, t) of a prompt is worth scores[w] + logits[w][t] - ln sum_i e^logits[w][i], and the best
 * `beams` of beams * vocab candidates become the new beams, best first, equal ones by rising w * vocab + t.  Sums and order are
 * in 64 bits; scores_out is rounded once.  A beam that `finished` marks (NULL: none; any nonzero byte) has the one
 * candidate (eos_token, scores[w]); a new beam is finished if its parent was or its token is eos_token (-1: no such
 * token; then finished must be NULL).  A NaN among logits or scores counts as -infinity, +infinity as the largest finite float; a first step
 * starts from scores 0, -infinity, -infinity, ..  beams <= 64, beams * vocab below 2^31.
 *
 * tokens, parents, scores_out, finished_out: `[prompts, beams]` (finished_out may be NULL).  lineage_out (NULL: none), `[prompts *
 * beams][lineage_capacity rounded up to 32]`: row i is the parent's row of `lineage` with i at position lens[parent], where
 * the new beam's next key and value go (slot i); lens `[prompts * beams]`, a position outside the row is left out.  Outputs may be the
 * corresponding inputs (lineage_out lineage, scores_out scores, finished_out finished) but overlap them no other way.  Uses the
 * library's per-stream scratch. */
int izwi_decode_beam_select_f32(const float* logits, int64_t prompts, int64_t beams, int64_t vocab, const float* scores,
                                const uint8_t* finished, int64_t eos_token, int32_t* tokens, int32_t* parents,
                                float* scores_out, uint8_t* finished_out, const uint8_t* lineage,
                                int64_t lineage_capacity, const int32_t* lens, uint8_t* lineage_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* IZWI_DECODE_OPS_H */
