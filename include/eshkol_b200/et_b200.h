/*
 * libet_b200 -- B200 (sm_100a) implementation of eshkol-transformer's f32
 * training-step hot path behind its K1 kernel ABI.
 *
 * Every entry point is plain C: pointers, sizes and the K1 v1 structs.  Each
 * declaration names the reference interface it replaces (path:line within the
 * eshkol-transformer project).  Device pointers are CUDA global memory on the
 * current device; "host" pointers are ordinary (preferably pinned) memory.
 * Functions returning int32_t return 0 on success or a K1 error category
 * (ET_KERNEL_ERROR_*) and fill the optional et_kernel_error record.
 */
#ifndef ESHKOL_B200_ET_B200_H
#define ESHKOL_B200_ET_B200_H

#include "eshkol_b200/kernel_abi_v1.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ET_B200_ABI_MAJOR 1u
#define ET_B200_ABI_MINOR 0u

/* ------------------------------------------------------------ library */

int32_t et_b200_abi_major_v1(void);
int32_t et_b200_abi_minor_v1(void);
/* Kernels this library has launched since load (all devices, all threads).
 * A caller samples it around a region to count the region's launches. */
uint64_t et_b200_launch_count_v1(void);
/* 0 when the current CUDA device is an sm_100 part this build runs on. */
int32_t et_b200_device_check_v1(et_kernel_error *error);

/* ------------------------------------------------------------ K1 providers
 *
 * Drop-in replacements for the reference's carrier-neutral providers.  They
 * accept dense zero-offset views on device "cuda" (device pointers, results
 * complete when invoke returns; the call first waits for all work already
 * enqueued on the device, so inputs produced on any stream are complete) and
 * on device "cpu" (host pointers, staged through the GPU).  Capabilities are
 * verified for every shape the kernels
 * support rather than the reference's exact tiny rows.  validate_call keeps
 * the reference's checks (finite inputs, canonical positions and masks, ids
 * in range) and its error categories; invoke_call never fails.
 */
/* replaces include/eshkol_transformer/a2_attention_abi.h:32
 * (kernel.causal-attention forward/backward, kernel.rope forward/backward) */
const et_kernel_provider_v1 *et_a2_kernel_provider_v1(void);
/* replaces include/eshkol_transformer/n2_primitives_abi.h:18
 * (kernel.matmul linear.*, kernel.norm, kernel.activation gelu/relu,
 *  kernel.residual, kernel.embedding-forward/backward) */
const et_kernel_provider_v1 *et_n2_kernel_provider_v1(void);
/* replaces include/eshkol_transformer/n3k_primitives_abi.h:12
 * (n3k.linear forward/backward-no-bias) */
const et_kernel_provider_v1 *et_n3k_kernel_provider_v1(void);
/* replaces include/eshkol_transformer/indexed_cross_entropy.h:22-29 */
int32_t et_l2_indexed_cross_entropy_abi_major_v1(void);
int32_t et_l2_indexed_cross_entropy_abi_minor_v1(void);
const et_kernel_provider_v1 *et_l2_indexed_cross_entropy_provider_v1(void);
/* Every capability above in one provider (sorted by name; each call goes to
 * the provider owning its capability), for K1 runtimes, which take exactly
 * one provider from their resolver (native/kernel_abi.c:764-840).  No
 * reference counterpart: the reference composes no providers. */
const et_kernel_provider_v1 *et_b200_kernel_provider_v1(void);
/* K2 capability facade support (native/k2_capabilities.c).  K2 discovers
 * through a fixed private resolver that answers only the K1 provider symbol
 * with its private context sentinel, and exact-audits the provider it gets,
 * identity by callback pointers (k2_capabilities.c:493-561).  These are that
 * resolver and that audit for the B200 provider: a K2 built over libet_b200
 * calls et_kernel_runtime_discover(et_b200_k2_resolver_v1,
 * (void *)et_b200_k2_resolver_context_v1(), ...) and admits the provider
 * when the audit returns ET_B200_K2_PROVIDER_EXACT (the values mirror
 * enum et_k2_provider_audit, k2_capabilities.c:565-570). */
enum {
  ET_B200_K2_PROVIDER_ABSENT = 0,
  ET_B200_K2_PROVIDER_VERSION_MISMATCH = 1,
  ET_B200_K2_PROVIDER_METADATA_MISMATCH = 2,
  ET_B200_K2_PROVIDER_EXACT = 3
};
const void *et_b200_k2_resolver_context_v1(void);
const et_kernel_provider_v1 *et_b200_k2_resolver_v1(void *context,
                                                    const char *symbol_name);
int32_t et_b200_k2_audit_provider_v1(const et_kernel_provider_v1 *provider);
/* Contraction mode (ET_B200_PRECISION_*) the kernel.matmul and n3k.linear
 * providers use; process-wide, default ET_B200_PRECISION_TF32X3.  No
 * reference counterpart: the reference's only mode is serial FP32. */
int32_t et_b200_k1_precision_v1(uint32_t precision);

/* ------------------------------------------------------------ attention on device
 * Causal attention with RoPE on device tensors, for callers that run many
 * steps without a K1 round trip per call (the A2 provider's arithmetic,
 * native/a2_attention_provider.c:669-790, with rope.forward on Q and K and
 * rope.backward on dQ and dK, :792-935).  No reference counterpart for the
 * split of the statistics: the forward returns per query row the maximum of
 * the scaled scores and the sum of their exponentials, which the backward
 * takes instead of recomputing the forward as a K1 backward call does.
 * Tensors are dense row-major f32 [batch, heads, len, head_dim] on the
 * current device; the calls enqueue on `stream` (a cudaStream_t, NULL = the
 * legacy default stream) and return without synchronising.  Inputs are not
 * validated on the device (finite values, canonical positions): the caller
 * supplies what the A2 provider's validate_call would accept. */
typedef struct et_b200_attention_v1 {
  size_t struct_size;
  int64_t batch, q_heads, kv_heads, q_len, k_len, head_dim;
  const int64_t *q_positions; /* device [batch, q_len], strictly increasing */
  const int64_t *k_positions; /* device [batch, k_len], strictly increasing */
  const uint8_t *keep;        /* device [batch, q_len, k_len] or NULL (all) */
  const float *rope_cos;      /* device [len, head_dim/2] (or [batch*len, ..]
                                 with rope_batched) for Q and K; NULL = no RoPE */
  const float *rope_sin;
  int32_t rope_batched;
  int32_t contraction; /* ET_B200_ATTENTION_* (0 = the default) */
} et_b200_attention_v1;
/* Contraction modes.  f32-grade (three products of operand pairs, about 22
 * significant bits per operand element):
 * ET_B200_ATTENTION_DEFAULT: binary16 pairs with per-tensor power-of-two
 *   scales at head_dim 128 and at head_dim 64 from q_len k_len = 768^2 up,
 *   3xTF32 pairs otherwise;
 * ET_B200_ATTENTION_BWD_PAIRS16: binary16 pairs in the backward at head_dim
 *   64 as well.
 * TF32-grade (one product of the hi parts, 11 significant bits per operand
 * element, the reference sweep's "TF32" mode):
 * ET_B200_ATTENTION_TF32: TF32 operands (round to nearest), binary16 ones
 *   with per-tensor scales (the same 11 bits) in the head_dim-128 backward. */
enum {
  ET_B200_ATTENTION_DEFAULT = 0,
  ET_B200_ATTENTION_BWD_PAIRS16 = 1,
  ET_B200_ATTENTION_TF32 = 2
};
/* Bytes of the workspace both calls take (256-byte aligned). */
size_t et_b200_attention_workspace_bytes_v1(const et_b200_attention_v1 *shape);
/* Host-side RoPE tables [len, head_dim/2] the way the reference builds its
 * rotation: inv_freq = (float)(1 / base^(2i/head_dim)), angle = (float)t *
 * inv_freq, cosf / sinf (a2_attention_provider.c:792-935 with the base-10000
 * frequencies the callers pass). */
void et_b200_rope_tables_v1(int64_t len, int64_t head_dim, double base,
                            float *cos_out, float *sin_out);
int32_t et_b200_attention_forward_v1(const et_b200_attention_v1 *shape,
                                     const float *q, const float *k,
                                     const float *v, float *o, float *row_max,
                                     float *row_sum, void *workspace,
                                     size_t workspace_bytes, void *stream,
                                     et_kernel_error *error);
/* workspace_from_forward: the workspace still holds what the forward of the
 * same Q/K/V wrote into it (the prepared operands are then reused). */
int32_t et_b200_attention_backward_v1(
    const et_b200_attention_v1 *shape, const float *q, const float *k,
    const float *v, const float *o, const float *dout, const float *row_max,
    const float *row_sum, float *dq, float *dk, float *dv, void *workspace,
    size_t workspace_bytes, int32_t workspace_from_forward, void *stream,
    et_kernel_error *error);

/* ------------------------------------------------------------ serving
 * Decoding for many requests at once on device tensors: appending keys and
 * values to a paged cache (the keys' RoPE applied on the way), causal
 * attention of the new tokens over it, and sampling the next token from
 * logits.  No reference counterpart: the reference caches one dense
 * [batch, kv_heads, capacity, head_dim] block per layer (the A2 KV cache
 * below) and leaves sampling to its host.  The arithmetic is the A2
 * provider's (native/a2_attention_provider.c:669-716, rope :792-935).
 * All calls enqueue on `stream` (a cudaStream_t, NULL = the legacy default
 * stream) of the current device, return without synchronising, allocate
 * nothing, keep nothing between calls and can be captured in a CUDA graph.
 * Pointers are device memory of the current device unless said otherwise. */
enum { ET_B200_DTYPE_F32 = 0, ET_B200_DTYPE_F16 = 1, ET_B200_DTYPE_BF16 = 2 };

/* Two pools of pages, one layer's keys and values, both addressed as element
 * page * page_stride + head * head_stride + slot * token_stride + d.  Any
 * page_size >= 1; head_dim a multiple of 8 up to 256; pools 16-byte aligned
 * and strides multiples of 16 bytes. */
typedef struct et_b200_paged_cache_v1 {
  size_t struct_size;
  void *keys;
  void *values;
  int64_t pages, page_size, kv_heads, head_dim;
  int64_t page_stride, head_stride, token_stride;
  uint32_t dtype; /* ET_B200_DTYPE_*, of the pools and of q, k, v and o */
  uint32_t reserved;
} et_b200_paged_cache_v1;

/* One step's requests.  Request b brings the rows offsets[b] .. offsets[b + 1]
 * - 1 of the token-major tensors as its last new tokens; lengths[b] counts
 * its tokens with them, so its token i of n stands at position lengths[b] - n
 * + i, in slot position % page_size of page page_table[b][position /
 * page_size].  A request may bring no token; a token at a negative position
 * is not stored and sees no key.  Rows of no request are not written, and
 * nothing depends on them.  max_new (the host's idea of the largest request)
 * only picks the kernel, and with it the roundings that the calls state for
 * few query rows and for many; max_length is not used so far.  The arrays are device
 * memory, read when the kernels run; what in them leads outside the pools or
 * tensors is not followed but recorded in *status (never cleared here): */
enum {
  ET_B200_PAGED_BAD_PAGE = 1,   /* a page outside the pool: reads as zeros,
                                   writes are dropped */
  ET_B200_PAGED_BAD_LENGTH = 2, /* a length below 0 or beyond the table's
                                   columns: clamped */
  ET_B200_PAGED_BAD_OFFSET = 4, /* offsets that fall or leave the tensors:
                                   clamped */
  ET_B200_PAGED_BAD_ROPE = 8,   /* a position beyond the RoPE tables: the last
                                   row is used */
  ET_B200_PAGED_TIMEOUT = 16    /* a kernel gave up waiting (some 2 s) for its
                                   own copies or products: o is not valid.
                                   Only the status word tells */
};
typedef struct et_b200_paged_batch_v1 {
  size_t struct_size;
  int64_t batch, tokens, table_columns;
  int64_t max_new, max_length;
  const int64_t *offsets;    /* [batch + 1], ascending from 0 */
  const int64_t *lengths;    /* [batch] */
  const int32_t *page_table; /* [batch, table_columns]; table_columns *
                                page_size < 2^31 - 4096 */
  int32_t *status;           /* one word, or NULL (then nothing of the above
                                is recorded, a timeout included) */
} et_b200_paged_batch_v1;

/* RoPE tables as et_b200_rope_tables_v1 lays them out: device f32 [rows,
 * head_dim / 2], indexed by position; both NULL = no rotation. */
typedef struct et_b200_paged_rope_v1 {
  const float *cos;
  const float *sin;
  int64_t rows;
} et_b200_paged_rope_v1;

/* Stores the step's keys (rotated) and values into their pages.  k and v:
 * [tokens, kv_heads, head_dim], heads dense, rows k_stride / v_stride elements
 * apart.  The rotation is computed in f32 and rounded once to the pools' type.
 * Two requests that own the same slot race. */
int32_t et_b200_paged_append_v1(const et_b200_paged_cache_v1 *cache,
                                const et_b200_paged_batch_v1 *batch,
                                const et_b200_paged_rope_v1 *rope,
                                const void *k, int64_t k_stride, const void *v,
                                int64_t v_stride, void *stream,
                                et_kernel_error *error);

/* o = softmax(q' k^T / sqrt(head_dim)) v over the keys at positions up to the
 * query's own (the new tokens' keys are in the cache already), q' = q rotated
 * in f32.  q and o: [tokens, q_heads, head_dim], heads dense, rows q_stride /
 * o_stride elements apart; q_heads a multiple of kv_heads up to 65,536, query
 * head h reads key head h / (q_heads / kv_heads).  A query that sees no key gets
 * zeros.
 * lse (f32 [tokens, q_heads], or NULL) receives ln(sum of exp of the scaled
 * scores), -inf without keys.  Scores, statistics and sums are f32; for the
 * tensor cores q' and the probabilities are rounded to the pools' type at f16
 * and bf16 (q' with its residual up to 16 query rows per kv head), and all
 * operands are carried as pairs of about 22 bits at f32 (above 16 query rows per
 * kv head elements more than 2^16 below their row's largest only to 2^-38 of
 * it).  Keys and values of positions below a request's length must be finite,
 * those hidden from a query included; slots behind may hold anything.  o must
 * overlap neither q nor the pools.  The workspace (any contents, overwritten; its
 * size does not depend on the batch) serves one call at a time: calls that may
 * overlap, and graphs that may, need one each. */
size_t et_b200_paged_attention_workspace_bytes_v1(
    const et_b200_paged_cache_v1 *cache, int64_t q_heads);
int32_t et_b200_paged_attention_v1(const et_b200_paged_cache_v1 *cache,
                                   const et_b200_paged_batch_v1 *batch,
                                   const et_b200_paged_rope_v1 *rope,
                                   int64_t q_heads, const void *q,
                                   int64_t q_stride, void *o, int64_t o_stride,
                                   float *lse, void *workspace,
                                   size_t workspace_bytes, void *stream,
                                   et_kernel_error *error);

/* A paged cache of 8 bits: as et_b200_paged_cache_v1, but an element is a byte of
 * type e4m3 (sign, 4 bits of exponent, 3 of fraction, largest 448; strides count
 * bytes and are multiples of 16, head_dim a multiple of 16 up to 256), and each
 * row of head_dim elements stands for its values times one f32 scale, at page *
 * scale_page_stride + head * scale_head_stride + slot * scale_token_stride of the
 * scale pools (in floats).  dtype is that of k, v, q and o.  A cached token and
 * head takes head_dim + 4 bytes of keys and as many of values. */
typedef struct et_b200_paged_cache8_v1 {
  size_t struct_size;
  void *keys;
  void *values;
  float *key_scales;
  float *value_scales;
  int64_t pages, page_size, kv_heads, head_dim;
  int64_t page_stride, head_stride, token_stride;
  int64_t scale_page_stride, scale_head_stride, scale_token_stride;
  uint32_t dtype; /* ET_B200_DTYPE_*, of k, v, q and o */
  uint32_t reserved;
} et_b200_paged_cache8_v1;

/* et_b200_paged_append_v1 into a cache of 8 bits: of each row x (a token's head; of
 * the keys rotated in f32) the scale s is the least power of two with |x| <= 448 s
 * for every element (no less than 2^-126; 0 for a row of zeros), and the stored
 * elements are x / s rounded to the nearest, ties to even.  A row that holds an
 * infinity or a NaN gets the scale NaN and elements of 0.  Two requests that own the
 * same slot race. */
int32_t et_b200_paged_append8_v1(const et_b200_paged_cache8_v1 *cache,
                                 const et_b200_paged_batch_v1 *batch,
                                 const et_b200_paged_rope_v1 *rope,
                                 const void *k, int64_t k_stride, const void *v,
                                 int64_t v_stride, void *stream,
                                 et_kernel_error *error);

/* et_b200_paged_attention_v1 over a cache of 8 bits, by the same rules but for these.
 * Finite scales are at most 2^126.  A row whose keys' or values' scale is not
 * finite makes NaN of o for every query that sees it (whose lse is then
 * unspecified) and of no other; elements must not be NaN, those hidden from a query
 * included.
 * Precision: scores, statistics and sums are f32.  q' is carried as binary16 of a
 * scale per row, at f32 and f16 with its residual (about 22 bits; at f16 not in the
 * chunks below); the probabilities as binary16, at f32 with their residual, in the
 * chunks below to no less than 2^-36 of a row's largest, else times their values'
 * scales and to no less than 2^-37 of the largest such product.
 * Elements and their products with scales that are powers of two (or 0), as the
 * append writes them, are exact.  Chunks (more than 48 query rows per kv head, as
 * max_new tells, at f32 up to 64 dims more than 64; head_dim up to 128) over pages of a
 * power of two of at least 8 slots whose scales lie side by side round other scales'
 * products to 11 bits; there, rows of a block of 128 keys (of the keys), or behind the
 * largest so far (of the values), whose scale is less than 2^-21 of the largest one's
 * lose bits. */
size_t et_b200_paged_attention8_workspace_bytes_v1(
    const et_b200_paged_cache8_v1 *cache, int64_t q_heads);
int32_t et_b200_paged_attention8_v1(const et_b200_paged_cache8_v1 *cache,
                                    const et_b200_paged_batch_v1 *batch,
                                    const et_b200_paged_rope_v1 *rope,
                                    int64_t q_heads, const void *q,
                                    int64_t q_stride, void *o, int64_t o_stride,
                                    float *lse, void *workspace,
                                    size_t workspace_bytes, void *stream,
                                    et_kernel_error *error);

/* Draws one token per row of logits [rows, vocabulary] (row_stride elements
 * apart) by inversion: with the weights w = exp((x - max x) / temperature) of
 * the tokens that the filters keep, ids[r] is the first token, in vocabulary
 * order, whose running sum of w exceeds uniform[r] times their total, and
 * logprobs[r] (or NULL) is ln(w / total) of it.  Filters, in this order, each
 * off where its array is NULL or its row's value says so; equal logits rank
 * by index, the most likely token is always kept:
 *   top_k  (<= 0: off)  the top_k most likely tokens;
 *   top_p  (>= 1: off)  tokens with less than top_p of the mass that top_k
 *                       left ranked before them;
 *   min_p  (<= 0: off)  w >= min_p (w of the most likely token is 1).
 * temperature NULL means 1; a row whose temperature is not above 2^-100 takes
 * the most likely token, with log-probability 0; at an infinite one every logit
 * above -inf weighs 1.  Weights are 2^-35 fixed point, so results depend on no
 * order of summation and tokens below 2^-36 of the likeliest weigh nothing.
 * -inf and NaN logits are never drawn; a row without others gets id -1 and
 * log-probability -inf; +inf logits share all weight.  vocabulary <= 2^22.
 * uniform is meant in [0, 1); other values act as the nearest end. */
typedef struct et_b200_sampling_v1 {
  size_t struct_size;
  int64_t rows, vocabulary, row_stride;
  uint32_t dtype; /* ET_B200_DTYPE_* of the logits */
  uint32_t reserved;
  const float *temperature; /* [rows] */
  const int64_t *top_k;     /* [rows] */
  const float *top_p;       /* [rows] */
  const float *min_p;       /* [rows] */
} et_b200_sampling_v1;
int32_t et_b200_sample_v1(const et_b200_sampling_v1 *shape, const void *logits,
                          const float *uniform, int64_t *ids, float *logprobs,
                          void *stream, et_kernel_error *error);

/* The distribution that et_b200_sample_v1 draws from, with the same shape and
 * filters: probs (f32 [rows, vocabulary], rows probs_stride floats apart) receives
 * w / total of every token that the filters keep and 0 for all others.  Weights
 * below 2^-36 of the likeliest count as 0, as there; others are f32 (not fixed
 * point) over a fixed-point total, so a probability, however small, is right to
 * 2^-21 + n 2^-36 of itself, n the number of kept tokens (the latter is 6e-5 where 2^22 are).  A
 * row that takes the most likely token gets a single 1, a row without a token to
 * draw only zeros.  probs must not overlap the logits. */
int32_t et_b200_probabilities_v1(const et_b200_sampling_v1 *shape,
                                 const void *logits, float *probs,
                                 int64_t probs_stride, void *stream,
                                 et_kernel_error *error);

/* Verification of drafted tokens (speculative decoding).  Request b's rows
 * offsets[b] .. offsets[b + 1] - 1 are the positions that one pass of the target
 * model gave: its last accepted token and the tokens drafted behind it, so row r
 * holds the target's distribution p_r (target [tokens, vocabulary], f32) of the
 * token that drafts[r] proposes; the last row of a request has no proposal
 * (drafts[r] is not read there).  draft (f32, rows as in target, or NULL) holds the
 * distributions q_r that the drafts were drawn from; NULL means drafts made without
 * chance (q_r is 1 at drafts[r]).  In order, a proposal x is accepted if
 * accept_uniform[r] q_r(x) < p_r(x); at the first that is not, the request's token
 * is drawn from max(p_r - q_r, 0), and behind its last accepted proposal from p_r of
 * the last row: the first token, in vocabulary order, whose running sum exceeds
 * draw_uniform[b] times the total.  Differences are f32, products
 * and sums are formed in 64 bits, in an order that depends on the vocabulary alone.
 * ids[r] receives the accepted proposals, then the drawn token, then -1 (ids may be
 * drafts); accepted[b] the number of accepted proposals (0 for a request without
 * rows).
 * Probabilities count as 0 where they are NaN or negative and as 1 above 1;
 * accept_uniform is meant in [0, 1) (a NaN accepts nothing), draw_uniform too
 * (other values act as the nearest end).  A proposal outside the vocabulary is
 * not accepted, and its q_r counts as 0 everywhere.  Where max(p - q, 0) is 0
 * everywhere the token is drawn from p; where that is too, it is -1.  Rows of no
 * request are not written.  offsets that fall or leave the tensors are clamped and
 * ET_B200_PAGED_BAD_OFFSET is recorded in *status.  Device memory throughout, read
 * when the kernel runs. */
typedef struct et_b200_verification_v1 {
  size_t struct_size;
  int64_t batch, tokens, vocabulary;
  int64_t target_stride, draft_stride; /* floats between rows */
  const int64_t *offsets;              /* [batch + 1], ascending from 0 */
  const int64_t *drafts;               /* [tokens] */
  const float *accept_uniform;         /* [tokens] */
  const float *draw_uniform;           /* [batch] */
  int32_t *status;                     /* one word, or NULL */
} et_b200_verification_v1;
int32_t et_b200_verify_v1(const et_b200_verification_v1 *shape,
                          const float *target, const float *draft, int64_t *ids,
                          int64_t *accepted, void *stream,
                          et_kernel_error *error);

/* ------------------------------------------------------------ synthetic data
 * Seeded inputs shared with the tests: value i of (seed, stream) is a pure
 * function of (seed, stream, i).  Host-only; no device is needed. */
void et_b200_fill_normal_v1(uint64_t seed, uint64_t stream, size_t count,
                            double mean, double stddev, float *out);
void et_b200_fill_tokens_v1(uint64_t seed, uint64_t stream, size_t count,
                            uint64_t vocabulary, int64_t *out);

/* ------------------------------------------------------------ O2 AdamW
 * Device counterpart of the O2 optimizer (native/o2_optimizer_internal.h:
 * 137-160 builder/step API; element maths o2_optimizer.c:1738-1756).  The
 * optimizer owns zero-initialised device moments; parameters and gradients are
 * caller-owned device tensors.  Each step divides gradients by the
 * normalisation weight, applies the global-L2 clip factor and the schedule
 * factor, and updates all tensors in one fused multi-tensor pass whose
 * per-element arithmetic is bit-identical to the reference. */
enum { ET_B200_O2_CLIP_NONE = 0, ET_B200_O2_CLIP_GLOBAL_L2 = 1 };
enum { ET_B200_O2_SCHEDULE_CONSTANT = 0, ET_B200_O2_SCHEDULE_LINEAR = 1 };

typedef struct et_b200_o2_parameter_v1 {
  size_t struct_size;
  float *value;    /* device, count f32 */
  float *gradient; /* device, count f32 (weighted numerators) */
  size_t count;
  uint32_t learning_rate_bits;
  uint32_t beta1_bits;
  uint32_t beta2_bits;
  uint32_t epsilon_bits;
  uint32_t weight_decay_bits;
  uint32_t reserved;
} et_b200_o2_parameter_v1;

typedef struct et_b200_o2_optimizer et_b200_o2_optimizer;

/* replaces et_o2_optimizer_builder_create_v1/_set_v1/_finish_v1
 * (native/o2_optimizer_internal.h:137-150) */
int32_t et_b200_o2_optimizer_create_v1(
    size_t parameter_count, const et_b200_o2_parameter_v1 *parameters,
    uint32_t clip_kind, uint32_t clip_max_bits, uint32_t schedule_kind,
    uint64_t warmup_updates, uint64_t total_updates,
    uint32_t minimum_ratio_bits, et_b200_o2_optimizer **optimizer,
    et_kernel_error *error);
/* replaces et_o2_optimizer_step_v1 (native/o2_optimizer.c:1784-1944).
 * normalization_weight_bits is the f32 bit pattern of the accumulated
 * contribution weight.  norm_bits (optional) receives the global norm.  All
 * or nothing like the reference's staged commit: a nonfinite gradient,
 * parameter or moment, or an update that would be nonfinite, leaves every
 * tensor and the update counter unchanged and returns INVALID_ARGUMENT.  The
 * global norm is an f64 sum of squares rounded once to f32; the reference's
 * is a scaled f32 recurrence in parameter order (o2_optimizer.c:1548-1618),
 * so the two norms (and with clipping active, the clipped updates) can differ
 * in the last bits. */
int32_t et_b200_o2_optimizer_step_v1(et_b200_o2_optimizer *optimizer,
                                     uint32_t normalization_weight_bits,
                                     uint32_t *norm_bits,
                                     et_kernel_error *error);
int32_t et_b200_o2_optimizer_completed_updates_v1(
    const et_b200_o2_optimizer *optimizer, uint64_t *updates);
/* Device pointers of parameter `index`'s moments (for checkpoint/inspection). */
int32_t et_b200_o2_optimizer_moments_v1(et_b200_o2_optimizer *optimizer,
                                        size_t index, float **exp_avg,
                                        float **exp_avg_sq);
void et_b200_o2_optimizer_destroy_v1(et_b200_o2_optimizer **optimizer);
/* AdamW step for callers that cannot allocate device memory: hosts that give
 * all of HBM to their own allocator at start-up, and loops that keep the
 * device footprint fixed because cudaMalloc/cudaFree can synchronise the
 * device mid-step.  No counterpart in the reference (its O2 optimizer is a
 * CPU object).  The caller owns the parameter, gradient and both moments
 * (device f32, `count` elements, moments zero before update 1); the call
 * divides the gradient by the normalisation weight, computes the global L2
 * norm, clips to clip_max_bits when that is nonzero, and applies the O2
 * update `update` (1-based, constant schedule) with the same per-element
 * rounding as et_b200_o2_optimizer_step_v1.  Its only scratch is a 64 KiB
 * file-scope device array that every GPU loading the library holds until
 * exit; count above ET_B200_ADAMW_NOALLOC_MAX_ELEMENTS is rejected.  Calls
 * share that array and its contents persist between calls: the call clears
 * what must start at zero itself, and calls that overlap on the GPU (on
 * different streams or host threads) race on it.  The first call on each
 * device looks up the array's device address (cudaGetSymbolAddress) and
 * should come before any stream capture.  Enqueued on `stream` (a
 * cudaStream_t, NULL = legacy default stream) and synchronised before
 * returning; norm_bits (optional) receives the norm.  The update is all or
 * nothing: a nonfinite gradient, a norm beyond f32's range, a nonfinite
 * parameter or moment, or an update that would produce a nonfinite value
 * leaves every tensor unchanged and returns INVALID_ARGUMENT (messages as
 * the reference's optimizer-step!). */
#define ET_B200_ADAMW_NOALLOC_MAX_ELEMENTS ((uint64_t)8192u * 65536u)
int32_t et_b200_adamw_step_noalloc_v1(
    float *value, const float *gradient, float *exp_avg, float *exp_avg_sq,
    uint64_t count, uint32_t learning_rate_bits, uint32_t beta1_bits,
    uint32_t beta2_bits, uint32_t epsilon_bits, uint32_t weight_decay_bits,
    uint64_t update, uint32_t normalization_weight_bits,
    uint32_t clip_max_bits, void *stream, uint32_t *norm_bits,
    et_kernel_error *error);
/* The schedule factor of update `update` as f32 bits: 1 for the constant
 * schedule; the exactly rounded linear warmup/decay ratio otherwise
 * (replaces et_o2_schedule_factor, native/o2_optimizer.c:1345-1374). */
uint32_t et_b200_o2_schedule_factor_v1(uint32_t kind, uint64_t warmup,
                                       uint64_t total,
                                       uint32_t minimum_ratio_bits,
                                       uint64_t update);

/* ------------------------------------------------------------ LM training
 * A decoder-only LM training step composed from the same primitives in the
 * reference's schedule order (native/m3_schedule.esk:3-52): token embedding,
 * L pre-LN blocks (fused QKV linear, RoPE on Q/K, causal attention, output
 * linear, residual, LN, FFN up, exact-erf GELU, FFN down, residual), final
 * LN, head tied to the embedding, indexed cross-entropy with the 1/N token
 * weight fused into its backward, AdamW.  This is the training loop's fast
 * path: it runs the kernels directly instead of one K1 dispatch per role.
 */
enum {
  ET_B200_PRECISION_TF32X3 = 0, /* 3xTF32 tcgen05 contractions (f32-grade) */
  ET_B200_PRECISION_TF32 = 1,   /* single TF32 tcgen05 contractions        */
  ET_B200_PRECISION_F32 = 2,    /* FP32 FFMA contractions (no tensor core)  */
  ET_B200_PRECISION_F16X3 = 3   /* split-f16 tcgen05 contractions: binary16
                                   hi/lo pairs with per-tensor power-of-two
                                   scales, 3 products (f32-grade)           */
};

typedef struct et_b200_lm_config_v1 {
  size_t struct_size;
  int64_t layers;
  int64_t d_model;
  int64_t heads;
  int64_t ffn;
  int64_t vocabulary;
  int64_t seq_len;
  int64_t batch;            /* sequences per step on this rank */
  int64_t global_tokens;    /* CE weight N across all ranks; 0 = batch*seq */
  uint32_t ln_epsilon_bits; /* 0x3727c5ac = 1e-5 */
  uint32_t precision;       /* ET_B200_PRECISION_* */
  double rope_base;         /* 10000 */
  uint32_t learning_rate_bits, beta1_bits, beta2_bits, epsilon_bits,
      weight_decay_bits;
  uint32_t reserved;
} et_b200_lm_config_v1;

typedef struct et_b200_lm et_b200_lm;

int32_t et_b200_lm_create_v1(const et_b200_lm_config_v1 *config,
                             et_b200_lm **lm, et_kernel_error *error);
void et_b200_lm_destroy_v1(et_b200_lm **lm);
/* Parameter tensors, in order, and their element counts. */
size_t et_b200_lm_tensor_count_v1(const et_b200_lm *lm);
size_t et_b200_lm_parameter_count_v1(const et_b200_lm *lm);
int32_t et_b200_lm_tensor_sizes_v1(const et_b200_lm *lm, size_t *sizes);
/* Seeded initialisation: weights N(0, 0.02), LN gammas 1, biases 0. */
int32_t et_b200_lm_init_v1(et_b200_lm *lm, uint64_t seed,
                           et_kernel_error *error);
/* which: 0 parameters, 1 gradients, 2 exp_avg, 3 exp_avg_sq (host copies). */
int32_t et_b200_lm_read_v1(et_b200_lm *lm, int32_t which, float *host,
                           size_t count, et_kernel_error *error);
int32_t et_b200_lm_write_v1(et_b200_lm *lm, int32_t which, const float *host,
                            size_t count, et_kernel_error *error);
/* One training step from HOST token ids/targets [batch, seq_len]: copies
 * them in, runs forward, backward (with the data-parallel gradient allreduce
 * when enabled), the AdamW update, and copies the mean loss out.  The update
 * is all or nothing, as O2's staged commit is (o2_optimizer.c:1813-1926): a
 * token id or target outside the vocabulary (on any rank), a nonfinite
 * gradient, parameter or moment, or an update that would be nonfinite leaves
 * parameters, moments and the update counter unchanged and returns
 * INVALID_ARGUMENT. */
int32_t et_b200_lm_step_v1(et_b200_lm *lm, const int64_t *host_ids,
                           const int64_t *host_targets, float *host_loss,
                           et_kernel_error *error);
/* The same step on DEVICE-resident ids/targets; the mean loss stays on the
 * device (device_loss may be NULL).  Enqueued on the model's stream; returns
 * without synchronising.  A step the host call above would reject is
 * skipped on the device with nothing updated; such steps are counted by
 * et_b200_lm_update_counts_v1 (the update number of later steps is taken
 * from the device's count of applied updates, so skipped steps do not shift
 * the bias corrections). */
int32_t et_b200_lm_step_device_v1(et_b200_lm *lm, const int64_t *device_ids,
                                  const int64_t *device_targets,
                                  float *device_loss, et_kernel_error *error);
/* Forward + backward only (no optimizer update): gradients left in place. */
int32_t et_b200_lm_forward_backward_v1(et_b200_lm *lm,
                                       const int64_t *host_ids,
                                       const int64_t *host_targets,
                                       float *host_loss,
                                       et_kernel_error *error);
/* Loss mask of the following steps (the L3S masked objective,
 * native/l3s_masked_objective_provider.c:125-175, with the reference's O2
 * division by the accumulated weight, o2_optimizer.c:1738): `mask` is
 * u8 [batch * seq_len] (row-major [batch, seq_len], the D2 loss-mask plane),
 * each byte 0 or 1, in host memory (on_device 0: checked and copied before
 * the call returns) or device memory (on_device 1: copied on the model's
 * stream; a byte other than 0 / 1 voids the next step, which then reports
 * INVALID_ARGUMENT with nothing updated).  NULL restores the unmasked
 * objective.  With a mask the loss is sum(mask ce) / sum(mask) over this
 * rank's tokens, each token's CE gradient is seeded with mask 2^-k
 * (k = ceil(log2 global tokens), an exact scaling) so the gradients hold the
 * mask-weighted numerators 2^-k, and AdamW divides them by the global weight
 * sum(mask) 2^-k (summed over the data-parallel ranks with the last gradient
 * bucket).  A step whose global weight is 0 updates nothing and reports
 * INVALID_ARGUMENT.  No reference counterpart for the entry point itself: the
 * reference feeds the mask through its Eshkol objective bridge. */
int32_t et_b200_lm_set_loss_mask_v1(et_b200_lm *lm, const uint8_t *mask,
                                    int32_t on_device, et_kernel_error *error);
/* The cudaStream_t the model enqueues on. */
void *et_b200_lm_stream_v1(et_b200_lm *lm);

/* ------------------------------------------------------------ D2 batch planes
 * The i64 input / target planes and the bool loss-mask plane of a fixed
 * [rows, seq_len] batch from one flat token stream, by the row rule of the
 * reference's D2 shard loader in packed mode (docs/D2_SHARD_LOADER.md, "Rows,
 * shift, mask, and ordering"): the stream holds 0 rows when length < 2, else
 * 1 + floor((length - 2) / seq_len); row r starts at r seq_len; a position
 * whose target exists in the stream takes input token[s + t], target
 * token[s + t + 1] and mask 1; every other position holds 0, 0, 0.  Host
 * memory; rows first_row .. first_row + rows - 1 of the stream (rows past its
 * end are all padding); INVALID_ARGUMENT when first_row is past the last row
 * (a batch needs a true mask bit).  Shuffling and shard boundaries (unpacked
 * mode) stay with the caller's loader. */
int64_t et_b200_d2_row_count_v1(uint64_t tokens, int64_t seq_len);
int32_t et_b200_d2_rows_v1(const int64_t *tokens, uint64_t length, int64_t seq_len,
                           int64_t first_row, int64_t rows, int64_t *ids,
                           int64_t *targets, uint8_t *mask, et_kernel_error *error);
/* Data parallelism: NCCL communicator over `world` ranks.  unique_id is the
 * 128-byte ncclUniqueId rank 0 obtained from et_b200_nccl_unique_id_v1 and
 * shared with every rank.  Gradients are then summed across ranks in buckets
 * on a side stream as backward produces them. */
int32_t et_b200_nccl_unique_id_v1(uint8_t unique_id[128],
                                  et_kernel_error *error);
int32_t et_b200_lm_enable_data_parallel_v1(et_b200_lm *lm,
                                           const uint8_t unique_id[128],
                                           int32_t rank, int32_t world,
                                           et_kernel_error *error);
/* Per-kernel-class timing with CUDA events on the model's stream.  Classes,
 * in order: 0 GEMM, 1 attention forward, 2 attention backward, 3 cross-
 * entropy, 4 AdamW (the writing pass), 5 LayerNorm, 6 other elementwise,
 * 7 embedding, 8 TF32 split, 9 allreduce wait, 10 AdamW check pass.  read
 * fills count >= 44 doubles: per class
 * {launch groups, milliseconds, algorithmic FLOP, algorithmic bytes}
 * accumulated since profiling was enabled; collect folds the events of
 * device-side steps into those totals (host steps do it themselves). */
int32_t et_b200_lm_profile_v1(et_b200_lm *lm, int32_t enable);
int32_t et_b200_lm_profile_collect_v1(et_b200_lm *lm);
int32_t et_b200_lm_profile_read_v1(et_b200_lm *lm, double *out, size_t count);
/* Split-f16 models (ET_B200_PRECISION_F16X3): how many steps of the
 * host-synchronised calls had an operand reach binary16's overflow and were
 * redone with 3xTF32 contractions since the model was created (0 for other
 * modes).  No reference counterpart: the reference has one contraction mode. */
int32_t et_b200_lm_f16_redone_steps_v1(const et_b200_lm *lm);
/* Applied AdamW updates (the reference's completed_updates,
 * o2_optimizer.c:1929) and device-enqueued steps whose update was skipped
 * since the model was created; synchronises the model's stream.  No
 * reference counterpart for `skipped`: reference steps are host calls that
 * return their error. */
int32_t et_b200_lm_update_counts_v1(et_b200_lm *lm, uint64_t *completed,
                                    uint64_t *skipped, et_kernel_error *error);

/* ------------------------------------------------------------ A2 KV cache
 *
 * The reference's transactional K/V cache with its storage in device memory
 * (replaces include/eshkol_transformer/a2_kv_cache.h:42-147, semantics of
 * native/a2_kv_cache.c:394-880).  Same names, arguments, lease rules and error
 * categories/codes.  Differences a caller sees: K/V storage [layers, batch,
 * kv_heads, capacity, head_dimension], the lengths [batch] and the key-keep
 * mask [batch, capacity] handed out by views and read borrows are device
 * ("cuda") tensor views on the GPU that was current at create; stage_layer
 * sources may be "cpu" or "cuda" views; append_counts stays a "cpu" view.
 * Every call has finished its device work when it returns.  The views feed
 * the A2 provider's attention directly (cached decoding: Tq new tokens over
 * Tk = capacity keys, the key-keep mask broadcast over the queries).
 */
typedef struct et_a2_kv_cache et_a2_kv_cache;
typedef struct et_a2_kv_cache_transaction et_a2_kv_cache_transaction;
typedef struct et_a2_kv_cache_transaction_view et_a2_kv_cache_transaction_view;
typedef struct et_a2_kv_cache_read_borrow et_a2_kv_cache_read_borrow;
/* replaces a2_kv_cache.h:42-53 */
int32_t et_a2_kv_cache_abi_major_v1(void);
int32_t et_a2_kv_cache_abi_minor_v1(void);
int32_t et_a2_kv_cache_abi_require_v1(uint32_t major, uint32_t minimum_minor,
                                      et_kernel_error *error);
/* replaces a2_kv_cache.h:61-68 (storage zero-initialised in device memory) */
int32_t et_a2_kv_cache_create_v1(uint64_t layers, uint64_t batch,
                                 uint64_t kv_heads, uint64_t capacity,
                                 uint64_t head_dimension,
                                 et_a2_kv_cache **cache,
                                 et_kernel_error *error);
int32_t et_a2_kv_cache_destroy_v1(et_a2_kv_cache **cache,
                                  et_kernel_error *error);
/* replaces a2_kv_cache.h:70-85 */
int32_t et_a2_kv_cache_transaction_begin_v1(
    et_a2_kv_cache *cache, uint64_t append_width,
    const et_kernel_tensor_view_v1 *append_counts,
    et_a2_kv_cache_transaction **transaction, et_kernel_error *error);
/* replaces a2_kv_cache.h:87-96 ("cpu" or "cuda" sources).  "cuda" sources
 * are read after a device synchronisation, so work that produced them on any
 * stream of that device (and was enqueued before this call) has finished;
 * work enqueued later, from another host thread, is not waited for. */
int32_t et_a2_kv_cache_transaction_stage_layer_v1(
    et_a2_kv_cache_transaction *transaction, uint64_t layer,
    const et_kernel_tensor_view_v1 *keys,
    const et_kernel_tensor_view_v1 *values, et_kernel_error *error);
/* replaces a2_kv_cache.h:98-120 (device views) */
int32_t et_a2_kv_cache_transaction_view_begin_v1(
    et_a2_kv_cache_transaction *transaction, uint64_t layer,
    et_a2_kv_cache_transaction_view **view, et_kernel_error *error);
int32_t et_a2_kv_cache_transaction_view_tensors_v1(
    const et_a2_kv_cache_transaction_view *view,
    const et_kernel_tensor_view_v1 **keys,
    const et_kernel_tensor_view_v1 **values,
    const et_kernel_tensor_view_v1 **effective_lengths,
    const et_kernel_tensor_view_v1 **key_keep_mask,
    et_kernel_error *error);
int32_t et_a2_kv_cache_transaction_view_end_v1(
    et_a2_kv_cache_transaction_view **view, et_kernel_error *error);
/* replaces a2_kv_cache.h:122-126 (abort scrubs staged slots to +0) */
int32_t et_a2_kv_cache_transaction_commit_v1(
    et_a2_kv_cache_transaction **transaction, et_kernel_error *error);
int32_t et_a2_kv_cache_transaction_abort_v1(
    et_a2_kv_cache_transaction **transaction, et_kernel_error *error);
/* replaces a2_kv_cache.h:128-147 (device views) */
int32_t et_a2_kv_cache_read_borrow_begin_v1(
    et_a2_kv_cache *cache, et_a2_kv_cache_read_borrow **borrow,
    et_kernel_error *error);
int32_t et_a2_kv_cache_read_borrow_layer_v1(
    et_a2_kv_cache_read_borrow *borrow, uint64_t layer,
    const et_kernel_tensor_view_v1 **keys,
    const et_kernel_tensor_view_v1 **values,
    const et_kernel_tensor_view_v1 **lengths,
    const et_kernel_tensor_view_v1 **key_keep_mask,
    et_kernel_error *error);
int32_t et_a2_kv_cache_read_borrow_end_v1(
    et_a2_kv_cache_read_borrow **borrow, et_kernel_error *error);

#ifdef __cplusplus
}
#endif

#include "eshkol_b200/o2_bridge.h"
#endif
