/*
 * qllama_model.h -- C ABI of the Llama model host around the attention path
 * (B200, sm_100a): the layers on either side of the attention operator, a
 * GGUF loader that puts the weights on the device, and the sampler.
 *
 * It replaces, for a device-resident model:
 *   Transformer::forward_with_cache   src/transformer/transformer.rs:238-266
 *   TransformerBlock::forward_with_cache  src/transformer/layers.rs:615-631
 *   Embedding / Linear / RmsNorm / Mlp  src/transformer/layers.rs:57-205, 538-579
 *   TensorOps::rms_norm / silu          src/tensor/ops.rs:96-136, 222-239
 *   Transformer::from_gguf, TransformerConfig::from_gguf
 *                                       src/transformer/transformer.rs:142-197,
 *                                       src/transformer/config.rs:71-164
 *   GgufFile::from_path / load_tensor   src/gguf/parser.rs:40-99, src/gguf/loader.rs:47-132
 *   generate (prefill, then one token per step)  src/main.rs:387-429
 *   Sampler::sample_slice               src/sampler/sampler.rs:119-325
 * The attention steps of each layer go through ql_attn_forward
 * (qllama_attn.h) on the caller's ql_kv.
 *
 * Conventions are those of qllama_attn.h: every entry point returns QL_OK or
 * a QL_ERR_* status with a message in ql_last_error(); validation happens
 * before device work; one host thread per context at a time.
 *
 * Arithmetic: weights and activations are f32.  Every matrix product keeps
 * the reference's order (one output element = a sequential f32 sum over the
 * inner dimension, each product rounded separately, no fused multiply-add);
 * RMSNorm sums squares in f64 in index order; SiLU evaluates exp in f64 and
 * rounds it to f32 (the correctly rounded single-precision exp; the
 * reference's libm expf is within 0.502 ulp, so about one value in a few
 * hundred differs in its last bit).  With an f32 KV cache the logits agree
 * with the reference's CPU path to about 1e-5, and bit for bit where the
 * host's SiLU rounds the same way; greedy tokens are identical.
 * Each layer's Q/K/V projections run fused with RoPE and the cache append
 * (ql_qkv_rope_append, below) for f32, f16 and bf16 caches.
 */
#ifndef QLLAMA_MODEL_H
#define QLLAMA_MODEL_H

#include <stdint.h>

#include "qllama_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* TransformerConfig (src/transformer/config.rs:12-31); head_dim =
 * hidden_size / num_heads. */
typedef struct {
  int32_t vocab_size;
  int32_t hidden_size;
  int32_t intermediate_size;
  int32_t num_heads;
  int32_t num_kv_heads;
  int32_t num_layers;
  int32_t max_position_embeddings;
  float rms_norm_eps;
  float rope_theta;
} ql_llama_config;

typedef struct ql_llama ql_llama;

/* Transformer::from_parts: allocates the device weights (zeros) and the
 * workspace for up to max_position_embeddings tokens per call.  The checks of
 * Attention::new / Mlp::new (layers.rs:244-286, 550-570) apply. */
int ql_llama_create(ql_ctx* ctx, const ql_llama_config* cfg, ql_llama** out);
int ql_llama_destroy(ql_llama* m);
int ql_llama_get_config(const ql_llama* m, ql_llama_config* out);

/* Sets one weight by its GGUF name (llama.cpp's LLM_TENSOR names, as
 * Transformer::from_gguf assembles them): token_embd.weight, output_norm.weight,
 * output.weight, blk.N.{attn_norm,attn_q,attn_k,attn_v,attn_output,ffn_norm,
 * ffn_gate,ffn_up,ffn_down}.weight.  `data` is host f32 in the reference's
 * logical layout after the GGUF dimension reversal: [out_features,
 * in_features] for projections, [vocab, hidden] for the embedding.  `n` must
 * equal the tensor's element count.  Without output.weight the lm_head shares
 * the embedding (tied embeddings, transformer.rs:150-155). */
int ql_llama_set_tensor(ql_llama* m, const char* name, const float* data, int64_t n);

/* GgufFile::from_path + Transformer::from_gguf: parses the file (GGUF v2/v3,
 * little-endian), derives the configuration from its metadata as
 * TransformerConfig::from_gguf does, and loads F32 and F16 tensors (F16
 * widened exactly to f32).  Quantised tensor types are rejected with the
 * reference's message ("not yet supported"). */
int ql_llama_load_gguf(ql_ctx* ctx, const char* path, ql_llama** out);

/* Transformer::forward_with_cache for sequence slot `seq` of `kv` (created
 * with the model's num_layers, num_kv_heads, head_dim; f32 storage keeps the
 * reference's arithmetic): ids [n] (host), logits [n, vocab] written to
 * `logits` (host or device memory as `mem` says; NULL computes only the
 * cache update).  start_pos must continue the cache (cache.rs:132-137) and
 * the last position must stay below max_position_embeddings
 * ("exceeds max_position_embeddings", transformer.rs:250-257). */
int ql_llama_forward(ql_llama* m, ql_kv* kv, int32_t seq, const int32_t* ids, int32_t n,
                     int64_t start_pos, float* logits, int32_t mem);

/* The projections fused with RoPE and the append: one launch computes the
 * Q, K and V projections of `x` (layers.rs:388-390), rotates q and k
 * (layers.rs:397-402, ops.rs:168-220) and writes K and V into the cache at the
 * call's positions (layers.rs:403-413, KvCache::update cache.rs:83-170).
 * args gives layer_idx, batch, new_len, seq_ids, start_pos, num_heads,
 * num_kv_heads, head_dim and rope_theta as for ql_attn_forward (q, k, v, out,
 * dtypes and mem are not read).  x: device f32 [batch*new_len, in_features];
 * wqkv_t: device f32 [in_features, (num_heads + 2*num_kv_heads)*head_dim],
 * the transposed weights of q, k and v side by side; q_rot: device f32
 * [batch, new_len, num_heads, head_dim], the rotated queries.  The cache
 * must store f32, f16 or bf16; positions must continue each sequence
 * ("must continue"), and the sequences' lengths advance.  Every product is an
 * f32 sequential sum in the reference's order. */
int ql_qkv_rope_append(ql_ctx* ctx, ql_kv* kv, const ql_attn_args* args, const float* x,
                       int32_t in_features, const float* wqkv_t, float* q_rot);

/* Steps 5-7 of forward_with_cache (layers.rs:425-455) over rows that
 * ql_qkv_rope_append has just written: args as for ql_attn_forward with
 * q = the rotated queries (in_dtype f32) and k, v unused; start_pos[b] +
 * new_len must equal the sequence's current length. */
int ql_attn_forward_appended(ql_ctx* ctx, ql_kv* kv, const ql_attn_args* args);

/* SamplerConfig (src/sampler/sampler.rs:15-25).  temperature <= 0 is greedy
 * (argmax after the repeat penalty, ties to the smaller id). */
typedef struct {
  float temperature;
  int32_t top_k;        /* 0 = no limit */
  float top_p;          /* >= 1 = no limit */
  float repeat_penalty; /* 1 = none */
} ql_sampler_config;

/* Sampler::sample_slice on the device for one row of logits: repeat penalty
 * over `context` (ids outside the vocabulary ignored, each id once), then
 * greedy argmax, or temperature, softmax (f64), top-k, top-p and the draw at
 * `r` (a uniform number in [0, 1) the caller supplies: the reference draws it
 * from its seeded generator, rng.gen::<f64>()).  logits [vocab] f32 and
 * context [n_context] int32 are device pointers; the token id is written to
 * the device int32 at token_out.  Invalid configurations are rejected as
 * SamplerConfig::validate does; a non-finite logit makes the kernel write -1
 * and raise the context's status (QL_ERR_DEVICE at the next synchronize). */
int ql_sample(ql_ctx* ctx, const float* logits, int32_t vocab, const int32_t* context,
              int32_t n_context, const ql_sampler_config* cfg, double r, int32_t* token_out);

/* generate() (src/main.rs:387-429) on the device: the prompt is prefilled at
 * position 0 of slot `seq`, then each step feeds back the sampled token.  The
 * whole loop is queued without a host round trip per step (the embedding of
 * a step reads the token the previous step's sampler wrote), unless eos_id >=
 * 0, in which case every step is checked and generation stops at EOS (not
 * counted, as in the reference).  `uniforms` holds one draw in [0, 1) per
 * step (NULL for greedy).  out_tokens (host, `steps` entries) receives the
 * generated ids, *n_out their count. */
int ql_llama_generate(ql_llama* m, ql_kv* kv, int32_t seq, const int32_t* prompt,
                      int32_t n_prompt, int32_t steps, int32_t eos_id,
                      const ql_sampler_config* cfg, const double* uniforms, int32_t* out_tokens,
                      int32_t* n_out);

/* ---- RMSNorm with the residual's addition, plain or 8-bit outputs ----------
 * Per row: s = x + residual (f32; s = x without a residual),
 *   y_i = s_i / sqrt(mean(s^2) + eps) * weight_i,
 * the norm of TransformerBlock::forward_with_cache (layers.rs:615-631) with
 * the residual's addition before it, in one pass, evaluated in f32 (the model
 * host's f32 path keeps the reference's f64 order instead).  sum_out receives
 * s rounded once to in_dtype; y is computed from the unrounded s.
 *
 * out_dtype F32, F16 or BF16: out [rows, hidden] holds y rounded once.
 * out_dtype Q8_0: out [rows, hidden] holds int8 values and out_scale
 * [rows, hidden/32] one f16 scale d per 32 columns, by the cache's rule:
 * d = max|y| / 127, value = round(y / d) with ties away from zero, d stored
 * as f16 (65504 at most; larger values saturate).  Quotients are f32 within some
 * units in the last place, so that a value within 1e-4 of a tie, or a d that close
 * (relative to f16's step) to one, may be the neighbouring one.  A block that holds a NaN or
 * an infinity gets a NaN scale, so that it reads back as NaN.
 *
 * x and residual have x_stride / residual_stride elements from row to row
 * (0 = hidden); sum_out, out and out_scale are contiguous.  sum_out may be x
 * or residual itself, and so may out, where the strides (and for out the types)
 * are the same; any other overlap of an output is refused.  Device pointers,
 * aligned to their element size. */
typedef struct {
  int32_t rows;          /* 0 is a no-op */
  int32_t hidden;        /* a multiple of 32 for Q8_0 */
  int32_t in_dtype;      /* x, residual, sum_out: F32, F16 or BF16 */
  int32_t weight_dtype;  /* F32, F16 or BF16 */
  int32_t out_dtype;     /* F32, F16, BF16 or Q8_0 */
  float eps;             /* finite, not negative */
  int64_t x_stride, residual_stride;
  const void* x;
  const void* residual;  /* may be NULL */
  const void* weight;    /* [hidden] */
  void* sum_out;         /* may be NULL; needs a residual */
  void* out;
  void* out_scale;       /* Q8_0 only */
} ql_norm_args;

int ql_rms_norm(ql_ctx* ctx, const ql_norm_args* args);

/* ---- 4-bit weights ----------------------------------------------------------
 * A weight matrix [out_features, in_features] of 4-bit codes with one f16
 * scale per row and `group` (32, 64 or 128) consecutive columns:
 *   w[n][k] = scale[n][k / group] * (code[n][k] - 8),  0 <= code <= 15.
 * Group 32 is GGUF's Q4_0.  The handle holds the matrix on the context's
 * device in the order the product kernel streams it (in_features is a
 * multiple of the group, at most 2^24; rows are padded to 16, columns to 64). */
typedef struct ql_q4 ql_q4;
int ql_q4_create(ql_ctx* ctx, int32_t out_features, int32_t in_features, int32_t group,
                 ql_q4** out);
/* Waits for the stream of the context that the handle was made with; products that
 * other contexts have queued must be done. */
int ql_q4_destroy(ql_q4* w);
int ql_q4_shape(const ql_q4* w, int32_t* out_features, int32_t* in_features, int32_t* group);
/* From codes [out_features, in_features/2] (byte j of a row: column 2j in the
 * low four bits, 2j+1 in the high ones) and f16 scales
 * [out_features, in_features/group].  mem: where both live.  From device
 * memory the copy is queued on the context's stream; from host memory the call
 * returns when it is done.  (The same holds for the two calls below.) */
int ql_q4_set(ql_q4* w, const uint8_t* codes, const void* scales, int32_t mem);
/* From GGUF Q4_0 blocks: in_features/32 blocks of 18 bytes per row (an f16
 * scale, then 16 bytes whose low bits are columns 0-15 and high bits columns
 * 16-31); `bytes` must be out_features * in_features/32 * 18.  Group 32 only. */
int ql_q4_set_blocks(ql_q4* w, const void* blocks, int64_t bytes, int32_t mem);
/* Quantises a dense matrix (F32, F16 or BF16, row_stride elements from row to
 * row, 0 = in_features): with m the group's value of largest magnitude (the
 * first of equals), scale = f16(m / -8) and
 * code = clamp(round(w / scale) + 8, 0, 15), ties to even; a group of zeros (or
 * whose scale underflows) gets scale 0, code 8.  A group that holds a NaN or an
 * infinity, or whose scale exceeds f16, gets a NaN scale. */
int ql_q4_quantize(ql_q4* w, const void* dense, int32_t dtype, int64_t row_stride, int32_t mem);
/* The codes and scales back, in ql_q4_set's layout (either may be NULL). */
int ql_q4_get(const ql_q4* w, uint8_t* codes, void* scales, int32_t mem);

/* y = x W^T for a few rows x [rows, in_features] (Linear::forward,
 * layers.rs:148-171): single tokens, drafted tokens, small batches.  The
 * kernel is built for a few rows, where the weights' bytes are the cost: a pass
 * over the weights takes up to 32 rows (F16, BF16, Q8_0) or 8 (F32), and more
 * rows are taken in that many passes.
 *   in_dtype F32, F16, BF16: x as given, every product with a code exact (an
 *     infinity in an F32 row gives NaN; F32 magnitudes below 2^-110 count in
 *     steps of 2^-133);
 *   in_dtype Q8_0: int8 values with x_scale [rows, in_features/32] f16, the
 *     output of ql_rms_norm (integer products, exact per block of 32).
 * Sums are f32; y [rows, out_features] is rounded once to out_dtype.  A row's
 * bits depend neither on the other rows' values nor on their number.  x_stride and y_stride are
 * elements from row to row (0 = contiguous); x_scale is contiguous.  y must not
 * overlap x.  Device pointers, aligned to their element size. */
typedef struct {
  int32_t rows;      /* 0 is a no-op */
  int32_t in_dtype;  /* F32, F16, BF16 or Q8_0 */
  int32_t out_dtype; /* F32, F16 or BF16 */
  int64_t x_stride, y_stride;
  const void* x;
  const void* x_scale; /* Q8_0 only */
  void* y;
} ql_linear_args;

int ql_linear_q4(ql_ctx* ctx, const ql_q4* w, const ql_linear_args* args);

/* Turns a model's projections and lm_head (its own or the tied embedding) into
 * 4-bit weights of `group` on the device and frees their f32 form; hidden_size
 * and intermediate_size must be multiples of the group.  From then on
 * ql_llama_forward and ql_llama_generate run ql_rms_norm (Q8_0) and ql_linear_q4
 * in place of the f32 kernels, and ql_llama_set_tensor is refused.  Logits then
 * differ from the reference's by the weights' and activations' rounding. */
int ql_llama_quantize(ql_llama* m, int32_t group);

/* ---- verification of drafted tokens -----------------------------------------
 * Speculative sampling for a batch of sequences: sequence b brings n_b drafted
 * tokens x_0 .. x_{n_b-1}, the target model's distributions p_0 .. p_{n_b} at
 * their positions and the one after them, and the distributions q_i that x_i was
 * drawn from.  Draft i is accepted while u_i * q_i(x_i) < p_i(x_i).  At the first
 * rejected draft a the new token is drawn from max(p_a - q_a, 0), normalised; if
 * none is rejected, a = n_b and it is drawn from p_a.  The draw at r = uniform
 * n_b takes the first token in id order whose running sum reaches r times the
 * whole, as ql_sample does.  Tokens so produced follow the target's distribution.
 *   tokens [batch, drafts + 1]: the accepted drafts, the new token, then -1
 *   accepted [batch]: a
 * form QL_VERIFY_LOGITS: p and q are softmax(logits / temperature); with
 * temperature <= 0 a draft is accepted while it is its row's largest logit (the
 * first of equals), and the new token is the largest of row a (the draft's logits
 * and the uniforms are not read).  Logits of -inf are probability 0.  A positive
 * temperature below f32's normal range (1.18e-38) is refused.
 * form QL_VERIFY_PROBS: target and draft hold the probabilities themselves, as
 * the caller's own filters left them (temperature is not read).
 * draft NULL: the drafts are certain (q_i(x_i) = 1), as those looked up in the
 * text are.  n_draft NULL: every sequence has `drafts`; entries are clamped to
 * [0, drafts], and what lies behind a sequence's drafts is not read.
 * Sums over the vocabulary that decide a token are f64, as are p_i(x_i) and q_i(x_i) in
 * a decision that f32 leaves open (below f64's smallest number they are 0); an id of
 * less than 1e-299 times its row's most probable counts as nothing in the sums.
 * A row that is reached and holds a NaN or +inf, or has no positive
 * probability, or a drafted id outside the vocabulary ends the sequence: its
 * new token is -1 and the context's status is raised (QL_ERR_DEVICE at the next
 * synchronize).  (Of probabilities, an accepted draft's rows are read at its id
 * alone.  Should the GPU not run a sequence's blocks side by side within a second, its
 * tokens are -1 and the status is raised too.)  ql_kv_truncate then drops the rejected drafts' cache rows.
 * tokens and accepted must not overlap each other or an input.  Device pointers,
 * aligned to their element size. */
#define QL_VERIFY_LOGITS 0
#define QL_VERIFY_PROBS 1
#define QL_VERIFY_MAX_DRAFTS 31
typedef struct {
  int32_t batch;       /* 0 is a no-op */
  int32_t drafts;      /* most drafted tokens of a sequence, 0 .. QL_VERIFY_MAX_DRAFTS */
  int32_t vocab;
  int32_t dtype;       /* target and draft: F32, F16 or BF16 */
  int32_t form;        /* QL_VERIFY_* */
  float temperature;
  int64_t target_stride, draft_stride; /* elements from row to row (0 = vocab) */
  const void* target;       /* [batch, drafts + 1, vocab] */
  const void* draft;        /* [batch, drafts, vocab] or NULL */
  const int32_t* draft_ids; /* [batch, drafts] */
  const int32_t* n_draft;   /* [batch] or NULL */
  const double* uniforms;   /* [batch, drafts + 1], each in [0, 1) */
  int32_t* tokens;
  int32_t* accepted;
} ql_verify_args;

int ql_verify_drafts(ql_ctx* ctx, const ql_verify_args* args);

#ifdef __cplusplus
}
#endif
#endif
