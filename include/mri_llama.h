/*
 * mri_llama.h — C ABI of the GPU LlamaModelInt8 (decoder layers, output
 * head and greedy decoding) built on the quantized-matmul entry points of
 * mri_qmatmul.h.
 *
 * Drop-in for src/model/llama/forward_int8.rs: LlamaModelInt8 (:416-546)
 * and TransformerBlockInt8 (:148-402), with the KvCache of
 * src/cache/kv_cache.rs.  All seven projections of every layer and the
 * output projection run through mri_matmul_int8_from_f32 (per-channel
 * INT8, as the reference), mri_matmul_q8_0_direct or
 * mri_matmul_q4_0_dequant, chosen per weight.
 *
 * Activations, logits, the KV cache and the embedding table live in device
 * memory; token ids passed to the forward calls are host values.  Calls are
 * asynchronous on `stream` (hipStream_t; NULL = default stream).  A model
 * handle keeps per-handle activation buffers: calls on one handle must be
 * ordered (one stream, or synchronized), like the reference's &mut self of
 * the cache they update.
 *
 * Numerics: projections as documented in mri_qmatmul.h; RoPE is bit-exact
 * given the reference's table (computed here on the host with the same
 * libm calls as RopeTable::new); RMSNorm, softmax, the attention value sum
 * and SwiGLU's exp agree with the reference to f32 rounding.
 */
#ifndef MRI_LLAMA_H
#define MRI_LLAMA_H

#include "mri_qmatmul.h"

#ifdef __cplusplus
extern "C" {
#endif

/* LlamaConfig fields the forward pass uses (src/model/llama/config.rs):
 * embedding_length, head_count, head_count_kv, feed_forward_length,
 * vocab_size, context_length (the RoPE table and cache length),
 * rms_norm_eps, rope_freq_base, block_count. */
typedef struct mri_llama_config {
    size_t dim;
    size_t n_heads;
    size_t n_kv_heads;
    size_t ffn_dim;
    size_t vocab;
    size_t max_seq;
    float eps;
    float rope_base;
    size_t n_layers;
} mri_llama_config;

typedef enum mri_weight_format {
    MRI_WEIGHT_INT8 = 0, /* const mri_qmatrix *       */
    MRI_WEIGHT_Q8_0 = 1, /* const mri_q8_0_matrix *   */
    MRI_WEIGHT_Q4_0 = 2, /* device pointer to raw Q4_0 blocks, n_out x k_in */
    /* const mri_q4_0_matrix *: Q4_0 weights projected with int8 activations
     * (mri_matmul_q4_0_w4a8, an extension without a reference counterpart) */
    MRI_WEIGHT_Q4_0_W4A8 = 3
} mri_weight_format;

/* A projection weight [n_out, k_in] (GGUF "out, in" layout).  The handle or
 * buffer is borrowed: it must outlive the model.  n_out / k_in are checked
 * against the role's shape. */
typedef struct mri_weight_ref {
    int format; /* mri_weight_format */
    const void *ptr;
    size_t n_out;
    size_t k_in;
} mri_weight_ref;

typedef struct mri_llama mri_llama;
typedef struct mri_kv_cache mri_kv_cache;

/* LlamaModelInt8::new, forward_int8.rs:430-444: token_embd [vocab, dim] and
 * output_norm [dim] are host f32 arrays (copied to the device); `output` is
 * the [vocab, dim] unembedding projection.  Layers are set with
 * mri_llama_set_layer before the first forward call.  InvalidShape for
 * inconsistent dimensions (n_heads % n_kv_heads, dim % n_heads, odd head
 * dim); Unsupported for a head dim other than 64 or 128. */
mri_status mri_llama_create(const mri_llama_config *cfg, const float *token_embd,
                            const float *output_norm, mri_weight_ref output,
                            mri_llama **out);
/* TransformerBlockInt8::new, forward_int8.rs:168-198: norms are host f32
 * [dim]; w[0..6] = wq [n_heads*hd, dim], wk, wv [n_kv*hd, dim],
 * wo [dim, n_heads*hd], wgate, wup [ffn, dim], wdown [dim, ffn].  When wq,
 * wk, wv (and wgate, wup) are handles of one format (INT8, Q8_0 or W4A8)
 * whose n_out are multiples of 16, the model builds owned row
 * concatenations of them here and projects once per group; outputs equal
 * the separate projections'.  Setting a layer again replaces them. */
mri_status mri_llama_set_layer(mri_llama *model, size_t layer, const float *attn_norm,
                               const float *ffn_norm, const mri_weight_ref w[7]);
void mri_llama_destroy(mri_llama *model);

/* KvCache::new, src/cache/kv_cache.rs:65: [n_layers][max_seq][n_kv*hd] f32
 * for K and V, zero-filled, on the device. */
mri_status mri_kv_cache_create(size_t n_layers, size_t max_seq, size_t n_kv_heads,
                               size_t head_dim, mri_kv_cache **out);
void mri_kv_cache_destroy(mri_kv_cache *cache);

/* Prefill of n tokens at positions start_pos .. start_pos + n - 1:
 * embed (forward_int8.rs:125-140), TransformerBlockInt8::forward_cached per
 * layer (:207-216, writing the cache), rmsnorm and the output projection
 * (:526-528).  logits: device [n, vocab].  InvalidShape for n == 0, a token
 * id >= vocab, or start_pos + n beyond the cache / RoPE table. */
mri_status mri_llama_forward_cached(mri_llama *model, const uint32_t *tokens, size_t n,
                                    size_t start_pos, mri_kv_cache *cache, float *logits,
                                    void *stream);
/* LlamaModelInt8::forward_decode, forward_int8.rs:538-546: one token at
 * position pos.  logits: device [vocab]. */
mri_status mri_llama_forward_decode(mri_llama *model, uint32_t token, size_t pos,
                                    mri_kv_cache *cache, float *logits, void *stream);
/* Greedy generation: forward_cached over the prompt (positions 0 ..), then
 * n_steps decode steps (positions n_prompt ..), each fed the argmax
 * (sampling/mod.rs:144-151, last of equal maxima) of the previous logits.
 * Token ids stay on the device between steps.  tokens_out (host,
 * n_steps + 1): the argmax of the prompt's last row, then of each step; it
 * is written when the call returns (the call synchronizes `stream`).
 * logits_out (device, nullable, [n_steps + 1, vocab]) receives the rows of
 * logits that chose them.  InvalidShape unless 1 <= n_prompt and
 * n_prompt + n_steps <= the cache / RoPE length. */
mri_status mri_llama_generate_greedy(mri_llama *model, const uint32_t *prompt, size_t n_prompt,
                                     size_t n_steps, mri_kv_cache *cache, uint32_t *tokens_out,
                                     float *logits_out, void *stream);

/* argmax of each of `rows` rows of n f32 values (device), as
 * sampling/mod.rs:144-151; idx: device [rows]. */
mri_status mri_argmax(const float *v, size_t rows, size_t n, uint32_t *idx, void *stream);

/* ===================================================================== */
/* A KV cache in 4-bit blocks for several sequences, and the operators of  */
/* a decode loop over it.  Extensions with no counterpart in the           */
/* reference, whose cache is f32 and holds one sequence                    */
/* (src/cache/kv_cache.rs), whose decoding is greedy                       */
/* (src/sampling/mod.rs:144-151) and which evicts nothing.  Device arrays  */
/* that are not aligned to 4 bytes are InvalidArgument.                    */
/* ===================================================================== */

/* Keys and values of n_layers layers and n_seqs sequences of up to max_seq
 * positions, in blocks of 32 consecutive dims of a head: an f16 scale d and
 * quants q in [-8, 7], 18 bytes.  With mx, mn the block's extremes and
 * a = mx if mx >= -mn else mn: d = f16(a / -8), saturated at +-65504,
 * q = clamp(rint(x / d), -8, 7) (exact quotients, ties to even; 0 where d is
 * 0); a block with a value that is not finite reads back as NaN.  A new cache
 * reads as zeros.  The handle is bound to the device it is created on; calls
 * with another current device are InvalidArgument.  It owns the workspace of
 * its attention calls (fixed at creation, so captured graphs hold it as long
 * as the handle lives): calls on one handle must be ordered, as on
 * mri_kv_cache; handles are independent.  No call allocates memory; calls of
 * more than 2^22 workgroups run in several launches.
 * InvalidShape for a zero size; Unsupported for a head dim other than 64 or
 * 128, or max_seq above 2^30. */
typedef struct mri_kv4_cache mri_kv4_cache;
mri_status mri_kv4_cache_create(size_t n_layers, size_t n_seqs, size_t max_seq,
                                size_t n_kv_heads, size_t head_dim, mri_kv4_cache **out);
/* Device bytes of the cached blocks and the workspace. */
size_t mri_kv4_cache_device_bytes(const mri_kv4_cache *cache);
void mri_kv4_cache_destroy(mri_kv4_cache *cache);

/* The rows of a call: `rows` per sequence for sequences first_seq ..
 * first_seq + n_seqs - 1.  Row i of the call's sequence b is at position
 * (pos ? pos[b] : start) + i.  pos and count are nullable DEVICE arrays
 * [n_seqs]; with count only the first min(count[b], rows) rows of a sequence
 * are real.  The other rows, and rows at positions >= max_seq, are neither
 * read nor written in any tensor.  (start + rows > max_seq without pos is
 * InvalidShape.) */
typedef struct mri_kv4_rows {
    size_t first_seq;
    size_t n_seqs;
    size_t rows;
    size_t start;
    const uint32_t *pos;
    const uint32_t *count;
} mri_kv4_rows;

/* Quantizes the rows' keys and values into the cache: k and v are
 * [n_seqs * rows] rows of n_kv_heads * head_dim f32, `stride` floats apart.
 * What the cache held at those positions is replaced. */
mri_status mri_kv4_append(mri_kv4_cache *cache, size_t layer, const mri_kv4_rows *rows,
                          const float *k, const float *v, size_t stride, void *stream);
/* The cached values at the rows' positions, as f32, of layers layer ..
 * layer + n_layers - 1: k and v are [n_layers][n_seqs * rows] rows, `stride`
 * floats apart. */
mri_status mri_kv4_read(const mri_kv4_cache *cache, size_t layer, size_t n_layers,
                        const mri_kv4_rows *rows, float *k, float *v, size_t stride,
                        void *stream);
/* Causal grouped-query attention over the cache: query row i of a sequence at
 * position p = pos + i sees keys 0 .. p (append first).  q and out are
 * [n_seqs * rows] rows of n_heads * head_dim f32, q_stride / out_stride
 * floats apart (out may be q, with equal strides, where weights is null); head
 * h reads KV head h / (n_heads / n_kv_heads).
 * InvalidShape when n_heads % n_kv_heads != 0; Unsupported for more than 2^20
 * heads, or rows * (n_heads / n_kv_heads) above 2^30.
 * weights (nullable): [cache n_seqs][n_kv_heads][max_seq] f32 of this layer,
 * the attention weight that each cached key has got: key t of a KV head gets
 * the sum of its probabilities over the call's rows and the head's query
 * heads, added to what was there for t < pos and stored for the new keys
 * t >= pos: a rejected draft's own entry is gone once its position is written
 * again.  What the rejected rows gave to the keys before them stays; weights of
 * accepted rows only take a call of their own after the verification, with
 * count = accepted + 1 (the call before it without weights).  The sums are in
 * a fixed order: equal calls give equal bits.
 * Outputs agree with f32 arithmetic on the cached values to f32 rounding, and,
 * for each key, to 2^-36 of the largest value that the call's rows see in the
 * same 32 dims of the head; of a query row, what is below 2^-39 of its largest
 * element is lost. */
mri_status mri_kv4_attend(mri_kv4_cache *cache, size_t layer, const mri_kv4_rows *rows,
                          const float *q, size_t q_stride, size_t n_heads, float *out,
                          size_t out_stride, float *weights, void *stream);
/* Eviction by accumulated weight, in every layer, sequence and KV head of
 * `src` by itself, into `dst` (a cache of the same sizes but its max_seq,
 * which holds at least `keep`; src itself: in place).  Sequence b holds
 * n = min(lens[b], src max_seq) keys.  If n <= keep all are kept; else the
 * last `recent` of them and, of the others, the keep - recent with the largest
 * weight (equal weights: the earlier key; NaN: below every number), in
 * the order they had.  dst holds them at positions 0 .., weights_out their
 * weights, kept their positions in src, lens_out[b] = min(n, keep).
 * Device arrays: weights [n_layers][n_seqs][n_kv_heads][src max_seq],
 * weights_out the same with dst's max_seq (in place: weights itself),
 * lens and lens_out [n_seqs] (may be the same array), kept [n_layers][n_seqs]
 * [n_kv_heads][keep], filled up with MRI_NO_TOKEN.  What dst and weights_out
 * hold past a sequence's keys stays.  The keys keep the rotation of their
 * original positions.  InvalidArgument for recent > keep, or weights_out ==
 * weights other than in place; InvalidShape for keep = 0 or caches that differ
 * or are too small. */
mri_status mri_kv4_evict(const mri_kv4_cache *src, mri_kv4_cache *dst, const float *weights,
                         float *weights_out, const uint32_t *lens, uint32_t *lens_out,
                         size_t keep, size_t recent, uint32_t *kept, void *stream);

/* mri_llama_forward_cached on sequence `seq` of a 4-bit cache: n tokens whose
 * rotary positions are start_pos .. and whose cache positions are cache_pos ..
 * (the same until keys are evicted).  Each row attends to the cached keys
 * before it, its own included.  weights (nullable): [n_layers][cache n_seqs]
 * [n_kv_heads][max_seq], added to as by mri_kv4_attend.  logits: device
 * [n, vocab].  Checks as mri_llama_forward_cached, for both position ranges. */
mri_status mri_llama_forward_kv4(mri_llama *model, const uint32_t *tokens, size_t n,
                                 size_t start_pos, mri_kv4_cache *cache, size_t seq,
                                 size_t cache_pos, float *weights, float *logits, void *stream);

/* Probabilities of rows of n logits (device, x_stride / out_stride floats
 * apart; out may be x): out = exp((x - max x) / temperature) / sum.  A row of
 * -inf only becomes zeros, one with NaN or +inf NaN.  Few rows of more than
 * 32768 logits are cut into parts, whose statistics pass through 256 KiB kept
 * per (device, stream), in two launches that no other thread's call on the
 * stream comes between; a call that is being captured uses none, takes longer
 * and gives the same bits.
 * InvalidArgument unless temperature > 0 and finite, or for x = out with
 * different strides; InvalidShape for n = 0 or a stride below n; Unsupported
 * for more than 2^21 rows. */
mri_status mri_softmax(const float *x, size_t rows, size_t n, size_t x_stride, float temperature,
                       float *out, size_t out_stride, void *stream);

/* Speculative verification: k drafted tokens a sequence against the target
 * model's probabilities.  Device arrays: drafts [n_seqs, k], target_probs
 * [n_seqs, k + 1, n], draft_probs [n_seqs, k, n] (nullable: the drafts were
 * not sampled, probability 1 each), uniforms [n_seqs, k + 1] in [0, 1),
 * n_drafts [n_seqs] (nullable: k; above k counts as k).
 * Draft i is accepted while uniforms[i] * q_i(draft) < p_i(draft) (exact).
 * With a of them accepted, one token more is drawn with uniforms[k]: from
 * max(p_a - q_a, 0) where a draft was rejected (from p_a where that has no
 * mass), from p_a where none was: the first token whose cumulative sum in f64 exceeds
 * uniforms[k] times the total.  accepted[b] = a; tokens [n_seqs, k + 1] = the
 * accepted drafts, the drawn token, then MRI_NO_TOKEN.  A draft id >= n is
 * rejected; where no token has a positive probability the drawn token is
 * MRI_NO_TOKEN.  A NaN target probability counts as 0; a token whose draft
 * probability is NaN is not accepted and has no part in the difference (where
 * that has no mass, p_a is drawn from with it).  InvalidShape
 * for n = 0; Unsupported for n = 2^32 - 1 and more, k above 2^20 or n_seqs
 * above 2^21. */
#define MRI_NO_TOKEN 0xffffffffu
mri_status mri_verify_drafts(const uint32_t *drafts, const float *draft_probs,
                             const float *target_probs, const float *uniforms,
                             const uint32_t *n_drafts, size_t n_seqs, size_t k, size_t n,
                             uint32_t *tokens, uint32_t *accepted, void *stream);

#ifdef __cplusplus
}
#endif
#endif
