/*
 * aether_ops.h — C ABI of the dense transformer ops on MI355X (gfx950).
 *
 * The reference's non-attention layers run these Metal kernels through its
 * Rust Ops engine:
 *   nexus-core/src/ops.metal:16-635   copy_buffer, embed_lookup, rms_norm, rope,
 *                                     matmul_f16, vecmat_f16, vecmat_scaled,
 *                                     silu_gate, add_residual, add_bias,
 *                                     matmul_scaled, causal_attention,
 *                                     multihead_attention, scale_f16
 *   nexus-core/src/ops.rs:166-462     the dispatch methods, called by
 *                                     InferenceEngine::forward_batch (inference.rs:456-634)
 * Each entry point below names the method it replaces and keeps its argument
 * order and meaning, with the engine first and a HIP stream last.  Pointers are
 * device pointers; f16 tensors are IEEE binary16 bit patterns (uint16_t).  The
 * calls are asynchronous on `hip_stream` (NULL is HIP's null stream): the
 * reference's batch mode (ops.rs:88-101, one command buffer per forward pass)
 * is a stream here, or a HIP graph captured from it.  A count of zero is a
 * no-op.  Every function returns AW_OK or a negative AW_E_* code of
 * aether_weaver.h, with the engine's last error describing the failure.
 *
 * Arithmetic is the reference's: f16 loads converted to fp32, fp32 sums and
 * products, one rounding to f16 (or fp32 for the scaled products) at the
 * store.  The products run on the matrix cores (v_mfma_f32_16x16x32_f16).
 */
#ifndef AETHER_OPS_H
#define AETHER_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "aether_weaver.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Ops::copy_buffer (ops.rs:166-180, ops.metal:16-26): dst[dst_off + i] =
 * src[src_off + i] for i < count; offsets in f16 elements.  The two ranges
 * must not overlap. */
int aw_ops_copy_buffer(aw_engine* engine, const uint16_t* src, uint16_t* dst, uint32_t count, uint32_t src_off,
                       uint32_t dst_off, void* hip_stream);

/* Ops::embed_lookup (ops.rs:183-206, ops.metal:33-49): output[t][:] =
 * embed_table[token_ids[t]][:] for t < seq_len, rows of hidden_size.  Added:
 * vocab_size, the table's row count.  An id >= vocab_size writes a zero row
 * and sets the engine's device error (aw_engine_check_device_errors reports
 * "token id"); the reference reads past its table. */
int aw_ops_embed_lookup(aw_engine* engine, const uint32_t* token_ids, const uint16_t* embed_table, uint16_t* output,
                        uint32_t hidden_size, uint32_t seq_len, uint32_t vocab_size, void* hip_stream);

/* Ops::rms_norm (ops.rs:209-231, ops.metal:59-99): per token row of
 * hidden_size, output = f16(x * (1 / sqrt(mean(x^2) + eps)) * weight).
 * output may equal input. */
int aw_ops_rms_norm(aw_engine* engine, const uint16_t* input, const uint16_t* weight, uint16_t* output,
                    uint32_t hidden_size, uint32_t num_tokens, float eps, void* hip_stream);

/* Ops::rope (ops.rs:234-263, ops.metal:107-155), in place on
 * q [num_tokens][q_heads][head_dim] and k [num_tokens][kv_heads][head_dim]:
 * the pair (x[p], x[p + head_dim/2]) of every head of token t rotates by
 * angle = f32(start_position + t) * freq_p, freq_p = 1 / theta^(2p / head_dim)
 * (taken in double precision and rounded to fp32; cos and sin of the fp32
 * angle likewise).  head_dim must be even; k may be NULL when kv_heads is 0. */
int aw_ops_rope(aw_engine* engine, uint16_t* q, uint16_t* k, uint32_t num_tokens, uint32_t q_heads, uint32_t kv_heads,
                uint32_t head_dim, uint32_t start_position, float theta, void* hip_stream);

/* Ops::matmul (ops.rs:266-296; kernels vecmat_f16 ops.metal:232-271 for m = 1,
 * matmul_f16 :170-216 otherwise): output [m][n] = f16(a [m][k] . b [n][k]^T),
 * fp32 accumulation.  Every column is computed (the reference's m = 1 launch
 * covers half of them: 8 columns per 256-thread group against the kernel's 16). */
int aw_ops_matmul(aw_engine* engine, const uint16_t* a, const uint16_t* b, uint16_t* output, uint32_t m, uint32_t n,
                  uint32_t k, void* hip_stream);

/* Ops::matmul_scaled (ops.rs:366-406; vecmat_scaled ops.metal:279-318,
 * matmul_scaled :380-422): output [m][n] = (a . b^T) * scale in fp32 (the
 * logits of the lm_head). */
int aw_ops_matmul_scaled(aw_engine* engine, const uint16_t* a, const uint16_t* b, float* output, uint32_t m,
                         uint32_t n, uint32_t k, float scale, void* hip_stream);

/* Ops::silu_gate (ops.rs:299-312, ops.metal:325-338):
 * output[i] = f16(gate[i] / (1 + exp(-gate[i])) * up[i]). */
int aw_ops_silu_gate(aw_engine* engine, const uint16_t* gate, const uint16_t* up, uint16_t* output, uint32_t size,
                     void* hip_stream);

/* Ops::add_residual (ops.rs:315-327, ops.metal:345-353): x[i] = f16(x[i] + residual[i]). */
int aw_ops_add_residual(aw_engine* engine, uint16_t* x, const uint16_t* residual, uint32_t size, void* hip_stream);

/* Ops::add_bias (ops.rs:330-343, ops.metal:360-371): x[t][d] = f16(x[t][d] + bias[d]). */
int aw_ops_add_bias(aw_engine* engine, uint16_t* x, const uint16_t* bias, uint32_t hidden_size, uint32_t num_tokens,
                    void* hip_stream);

/* Ops::scale_f16 (ops.rs:350-363, ops.metal:627-635): x[i] = f16(x[i] * scale). */
int aw_ops_scale_f16(aw_engine* engine, uint16_t* x, uint32_t count, float scale, void* hip_stream);

/* Ops::causal_attention (ops.rs:409-430, ops.metal:435-518), the legacy
 * single-head attention: output [head_dim] = softmax(q . K^T / sqrt(head_dim)) V
 * over kv_len rows of k and v [rows][head_dim].  Runs as
 * aw_multihead_attention_device with one head and one query, so head_dim is 64
 * or 128 and k and v must hold cache_tokens >= kv_len rounded up to 16 rows
 * (the reference's kv_len <= 4096 limit does not apply). */
int aw_ops_causal_attention(aw_engine* engine, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                            uint16_t* output, uint32_t kv_len, uint32_t head_dim, uint64_t cache_tokens,
                            void* hip_stream);

/* Ops::multihead_attention is aw_multihead_attention_device (aether_weaver.h). */

/* ---- fused forms (no reference counterpart) --------------------------------
 * Pairs and triples of the calls above that forward_batch makes back to back
 * (inference.rs:518-600), each in one launch, with the output bits of the
 * separate calls: a product's bits do not depend on how many products share a
 * launch (its K partial sums are added in a fixed order). */

/* aw_ops_matmul, aw_ops_scale_f16 of its output by residual_multiplier, then
 * aw_ops_add_residual of it into x (ops.rs:266-296, :350-363, :315-327; the
 * o_proj and down_proj steps, inference.rs:564-572,592-600):
 * p = f16(a . b^T), p = f16(p * residual_multiplier), x [m][n] = f16(x + p).
 * A multiplier of 1 (the reference skips the scale then) gives the same bits. */
int aw_ops_matmul_add_residual(aw_engine* engine, const uint16_t* a, const uint16_t* b, uint16_t* x, uint32_t m,
                               uint32_t n, uint32_t k, float residual_multiplier, void* hip_stream);

/* aw_ops_matmul with b_gate and with b_up, then aw_ops_silu_gate (ops.rs:266-312;
 * inference.rs:586-591): output [m][n] = f16(silu(f16(a . b_gate^T)) * f16(a . b_up^T)).
 * m <= 64 (decode and verify steps); larger m returns AW_E_UNSUPPORTED. */
int aw_ops_matmul_silu_gate(aw_engine* engine, const uint16_t* a, const uint16_t* b_gate, const uint16_t* b_up,
                            uint16_t* output, uint32_t m, uint32_t n, uint32_t k, void* hip_stream);

/* The three aw_ops_matmul calls of the q, k and v projections (inference.rs:518-523):
 * q [m][n_q] = a . b_q^T, k_out [m][n_kv] = a . b_k^T, v_out [m][n_kv] = a . b_v^T. */
int aw_ops_matmul_qkv(aw_engine* engine, const uint16_t* a, const uint16_t* b_q, const uint16_t* b_k,
                      const uint16_t* b_v, uint16_t* q, uint16_t* k_out, uint16_t* v_out, uint32_t m, uint32_t n_q,
                      uint32_t n_kv, uint32_t k, void* hip_stream);

/* ---- rotary positions, head norms, paged appends (no reference counterpart) ---
 * What a batch over pages needs around aw_decode_device that aw_ops_rope and
 * aw_ops_copy_buffer do not give: a position for each token, either order of
 * pairs, part of a head, frequencies scaled for long contexts, rows that are
 * views of a fused q/k/v product, each head normed first, and the rows written
 * through the block table. */

#define AW_ROTARY_HALF        0u /* pair p is dims (p, p + rotary_dim / 2), as aw_ops_rope's */
#define AW_ROTARY_INTERLEAVED 1u /* pair p is dims (2 p, 2 p + 1) */

#define AW_ROTARY_SCALE_NONE   0u /* f_p = theta^(-2 p / rotary_dim) */
#define AW_ROTARY_SCALE_LINEAR 1u /* f_p / factor (position interpolation) */
#define AW_ROTARY_SCALE_NTK    2u /* theta * factor^(rotary_dim / (rotary_dim - 2)) for theta; rotary_dim > 2 */
#define AW_ROTARY_SCALE_PARTS  3u /* (1 - g) f_p / factor + g f_p with g = clamp((r_p - low) / (high - low), 0, 1),
                                     r_p = original_length * f_p / (2 pi) the pair's turns over that length: pairs
                                     that turn often are kept, those that turn less than `low` times interpolated.
                                     The ramp is over turns; models whose ramp is over the pair's index, between
                                     rounded bounds, pass frequencies of their own as inv_freq */

typedef struct aw_rotary_scaling {
    uint32_t rotary_dim, kind;            /* AW_ROTARY_SCALE_* */
    double theta, factor;                 /* factor: unused by NONE */
    double original_length, low, high;    /* PARTS; 0 <= low < high */
} aw_rotary_scaling;

/* Host only: the rotary_dim / 2 frequencies, in radians per position, into
 * `inv_freq` (host memory). */
int aw_rotary_frequencies(const aw_rotary_scaling* scaling, double* inv_freq);

/* One call's rows.  Strides are in f16 elements from token to token, 0 for heads *
 * head_dim; the heads of a token are contiguous.  Rows of any alignment are taken.
 * Rows, frequencies, positions and weights are device memory. */
typedef struct aw_rotary_desc {
    uint32_t num_tokens, q_heads, kv_heads, head_dim; /* <= 2^24 tokens; head_dim <= 1024; either head count may be 0 */
    uint32_t rotary_dim;            /* even, <= head_dim: dims [0, rotary_dim) turn, the others pass */
    uint32_t layout;                /* AW_ROTARY_HALF or AW_ROTARY_INTERLEAVED */
    uint32_t start_position;        /* of token 0, where positions is NULL; positions are taken modulo 2^32 */
    float    magnitude;             /* cosines and sines are multiplied by it (1: a plain rotation) */
    float    eps;                   /* aw_ops_qk_norm_rotary and appends with norms */
    uint32_t reserved;              /* 0 */
    uint64_t q_stride, k_stride, q_out_stride, k_out_stride;
    const uint16_t* q;              /* [num_tokens][q_heads][head_dim] */
    const uint16_t* k;              /* [num_tokens][kv_heads][head_dim] */
    uint16_t*       q_out;          /* may be q (same stride: in place); shares no element with other rows */
    uint16_t*       k_out;          /* likewise k; NULL in an append */
    const uint16_t* q_norm;         /* [head_dim] weights */
    const uint16_t* k_norm;
    const uint32_t* positions;      /* [num_tokens], or NULL: start_position + token */
    const double*   inv_freq;       /* [rotary_dim / 2] */
} aw_rotary_desc;

/* Pair (x0, x1) of every head of token t becomes magnitude * (x0 cos a - x1 sin a,
 * x0 sin a + x1 cos a), a = position * inv_freq[p] taken in 64 bits (aw_ops_rope: in
 * 32); cos, sin and the products in fp32, one rounding at the store.  Dims past
 * rotary_dim are copied.  q_norm and k_norm must be NULL. */
int aw_ops_rotary(aw_engine* engine, const aw_rotary_desc* desc, void* hip_stream);

/* x * (1 / sqrt(mean(x^2) + eps)) * weight over each head's head_dim (fp32, as
 * aw_ops_rms_norm), then aw_ops_rotary of it without rounding in between.  Needs the
 * weights of every kind of head it is given; rotary_dim may be 0 (norms alone). */
int aw_ops_qk_norm_rotary(aw_engine* engine, const aw_rotary_desc* desc, void* hip_stream);

/* New tokens of `batch` sequences into their pages: k (normed where k_norm is given,
 * turned where rotary_dim > 0) and v into the rows that the block table names, q
 * (likewise) into q_out.  The table and the counts are those of the
 * aw_decode_device call that follows (AW_F_SEQ_HOT_TOKENS): refs [batch][refs_stride],
 * of which a sequence's first hot_count entries are its hot pages, and seq_hot
 * [batch], the tokens of each sequence AFTER the append.  Sequence b's new tokens are
 * rows token_offsets[b] .. token_offsets[b + 1] - 1 (token_offsets [batch + 1],
 * ascending, from 0; NULL: num_tokens / batch rows each); the last of them is token
 * seq_hot[b] - 1.  Their rotary position is start_position + that place, or
 * rows.positions.  For rows behind the last sequence (a padded batch)
 * nothing is written.  A page index past hot_count or a ref past hot_blocks
 * sets the device error "hot block ref": that token's k and v are not written.  A
 * sequence with more new tokens than seq_hot, or offsets that descend, set "sequence
 * length": nothing of those tokens is written (aw_engine_check_device_errors).  Two
 * tokens must not share a row of the pools: which is kept is then undefined.  The pools
 * overlap neither each other nor the rows. */
typedef struct aw_append_desc {
    aw_rotary_desc rows;            /* k_out NULL; q may be absent (q_heads 0) */
    uint32_t batch, hot_count, refs_stride, reserved; /* batch <= 2^24 */
    uint64_t v_stride, hot_blocks;
    const uint16_t* v;              /* [num_tokens][kv_heads][head_dim], NULL with hot_v */
    uint16_t* hot_k;                /* [hot_blocks][16][kv_heads][head_dim] */
    uint16_t* hot_v;                /* likewise, or NULL: the K row is the value (aw_decode_desc) */
    const uint32_t* refs;
    const uint32_t* seq_hot;
    const uint32_t* token_offsets;
} aw_append_desc;

int aw_ops_append_paged(aw_engine* engine, const aw_append_desc* desc, void* hip_stream);

/* The host checks of the calls above (aw_ops_qk_norm_rotary's where `norms` is not 0),
 * without an engine or a GPU: AW_OK or the code that the call returns, and its text in
 * `msg` (may be NULL).  What the tables and counts in device memory hold is checked by
 * the kernel alone. */
int aw_ops_check_rotary(const aw_rotary_desc* desc, int norms, char* msg, size_t msg_len);
int aw_ops_check_append(const aw_append_desc* desc, char* msg, size_t msg_len);

/* sizeof(aw_rotary_scaling), sizeof(aw_rotary_desc), sizeof(aw_append_desc), for bindings. */
void aw_abi_ops_desc_sizes(size_t sizes[3]);

/* ---- a step over trees of drafted tokens (no reference counterpart) ------------
 * The reference drafts a chain and verifies it on the host (nexus-core/src/agent.rs:337-410).
 * Here each sequence of a batch has a tree of `nodes` to verify: node 0 is its newest
 * token, every other node continues its parent, an earlier node.  One step of the model
 * checks all of them without the host in between:
 *   aw_ops_page_tables            offsets, pages, slots, positions and the tree's mask, from the lengths
 *   (products, aw_ops_rotary with those positions)
 *   aw_tree_attention_device      each node over the sequence's pages, its ancestors and itself (aether_weaver.h)
 *   (products, aw_ops_matmul_scaled)
 *   aw_ops_adjust_logits          penalties, biases, grammar masks, the best token of each row
 *   aw_ops_accept_tree            the path that the target's tokens take, its rows into the pages
 * Rows are flat: sequence b's nodes are rows token_offsets[b] .. token_offsets[b + 1] - 1
 * (token_offsets [batch + 1], ascending, from 0; NULL: num_tokens / batch rows each).  Rows
 * behind the last sequence (a padded batch) belong to none.  A tree's mask is
 * [num_tokens][mask_words] words: bit j of row i (bit j % 32 of word j / 32) says that node i
 * sees node j of its own sequence.  Device pointers; outputs overlap neither inputs nor each
 * other (but where a call says so).  Tokens and lengths out of range set the engine's device error
 * (aw_engine_check_device_errors) and are taken as stated. */

#define AW_MAX_NODES 1024u /* nodes of a sequence's tree: 32 mask words */
#define AW_NO_SLOT INT64_MIN /* the slot of a token that there was no page for */

/* Per sequence: seq_held tokens in pages before the step, seq_new new ones (nodes), seq_pages
 * entries of its row of refs that name pages (NULL: as many as its tokens need; more where an
 * earlier step left pages unfilled).  Where held + new tokens need more, the row is
 * continued with free_pages[f], free_pages[f + 1], .., in the order of the sequences, f =
 * *free_first (NULL: 0).  Outputs, each but refs, seq_hot and token_offsets may be NULL:
 *   refs          [batch][refs_stride], its new entries alone; seq_pages + the pages taken in pages_out
 *   seq_hot       held + new (what aw_ops_append_paged takes)
 *   token_offsets [batch + 1]
 *   free_next     [1] the place in free_pages behind the last page taken
 *   slots         [num_tokens] the row of the pools of each new token, ref * 16 + place % 16, or AW_NO_SLOT
 *   positions     [num_tokens] its place; with parents: held + its depth in the tree
 *   tree_mask     [num_tokens][mask_words], required with parents: itself and its ancestors
 * parents [num_tokens]: node numbers within the tree, < 0 for a root; one that is not an earlier node
 * sets "sequence length" and makes a root.  Rows behind the last sequence: slot -1, position 0,
 * mask 0.  A sequence has seq_new rows whatever else is wrong with it (fewer where num_tokens end, which sets
 * "sequence length"), so none moves the rows of those behind it.  Its new tokens past hot_count pages,
 * all of them where seq_held needs more pages than seq_pages or (with parents) there are more than 32
 * mask_words, set "sequence length" and take no page; those that free_pages has none for set "free pages".
 * Each such token gets AW_NO_SLOT, and its entry, where it lies within hot_count and behind seq_pages,
 * 0x7FFFFFFF (refused by the calls that read it), which is not counted in pages_out: a later step with
 * seq_held up to 16 * pages_out takes a page for it.  One of the seq_pages entries that is 0x7FFFFFFF sets
 * "free pages" where a new token falls into it.  A node past 32 mask_words sees nothing, at position held. */
typedef struct aw_tables_desc {
    uint32_t batch, num_tokens;          /* batch <= 2^20, num_tokens <= 2^24 */
    uint32_t hot_count, refs_stride;     /* entries of a row, <= 2^26; refs_stride >= hot_count */
    uint32_t free_count, mask_words;     /* free_count <= 2^30; mask_words <= 32, 0 without parents */
    const uint32_t* seq_held;
    const uint32_t* seq_new;
    const uint32_t* seq_pages;
    const uint32_t* free_pages;          /* [free_count] */
    const uint32_t* free_first;
    const int32_t*  parents;
    uint32_t* refs;
    uint32_t* seq_hot;
    uint32_t* pages_out;
    uint32_t* token_offsets;
    uint32_t* free_next;
    int64_t*  slots;
    uint32_t* positions;
    uint32_t* tree_mask;
} aw_tables_desc;

int aw_ops_page_tables(aw_engine* engine, const aw_tables_desc* desc, void* hip_stream);

#define AW_LOGITS_F16 1u /* logits and out are f16, else fp32 */

/* Rows of logits before a token is chosen.  With c the times that token v stands among the
 * sequence's history behind its first prompt_count tokens and among the tokens of the
 * nodes that the row's mask names, and `seen` where c > 0 or v is in the prompt, in fp32, each step rounded:
 *   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
 *   x = x - frequency * c;  c > 0: x = x - presence
 *   x = x + bias of v;  v not allowed: x = -inf
 * out (f16: rounded once; may be logits; NULL: best alone) and best, the lowest of the tokens of
 * the largest x in fp32, -1 where no x is above -inf (a NaN is never the largest; NULL: none).
 * history [batch][history_stride], of which history_count[b] tokens count (and bias_ids and
 * bias_values [batch][bias_stride], bias_count); where bias_ids names a token twice the last entry
 * holds.  allowed: bits [allowed_rows][allowed_stride words], 1 for a token that may follow; row t
 * takes allowed row allowed_index[t], none where that is negative (NULL: row t); an index
 * >= allowed_rows sets "token id" and allows nothing.  History, bias and node tokens >= vocab_size
 * are passed over.  Each of the penalties, and each group of pointers, may be NULL.  Counts past their
 * stride are taken as it and set "sequence length".  So do token_offsets that do not begin at 0, descend or pass
 * num_tokens, and rows of any sequence may then be left as they were. */
typedef struct aw_logits_desc {
    uint32_t num_tokens, vocab_size;     /* rows <= 2^24, vocab_size <= 2^24 */
    uint32_t batch, flags;               /* batch <= 2^20; 0 or AW_LOGITS_F16 */
    uint32_t mask_words;                 /* <= 32, 0 without nodes */
    uint32_t history_stride;             /* <= 2^20 */
    uint32_t bias_stride;                /* <= 1023 */
    uint32_t allowed_rows;
    uint64_t logits_stride, out_stride;  /* elements from row to row, 0 for vocab_size */
    uint64_t allowed_stride;             /* words, 0 for ceil(vocab_size / 32) */
    const void* logits;                  /* at their elements' alignment */
    void*       out;
    int32_t*    best;                    /* [num_tokens] */
    const uint32_t* token_offsets;
    const uint32_t* history;
    const uint32_t* history_count;
    const uint32_t* prompt_count;        /* NULL: 0 each */
    const float* repetition;             /* [batch] each */
    const float* frequency;
    const float* presence;
    const uint32_t* node_tokens;         /* [num_tokens], with tree_mask */
    const uint32_t* tree_mask;
    const uint32_t* bias_ids;
    const float*    bias_values;
    const uint32_t* bias_count;
    const uint32_t* allowed;
    const int32_t*  allowed_index;
} aw_logits_desc;

/* `best` takes scratch of the engine's workspace, 8 bytes a row and 1024 tokens or more, as in
 * aw_decode_device, also under capture. */
int aw_ops_adjust_logits(aw_engine* engine, const aw_logits_desc* desc, void* hip_stream);

/* From node 0 of each tree, whose token is kept, on: of the children of the node kept last
 * the lowest whose token is targets[that node] is kept too, until there is none (a target of
 * 0xFFFFFFFF, a best of -1, is no token).  Where slots are given a path ends before its j-th node if the
 * sequence's j-th row has AW_NO_SLOT: a later step, with a page for it, takes that token again.
 *   accepted   [batch] how many are kept (0 for a sequence without nodes, or without a page for node 0)
 *   next_token [batch] targets[the last one kept] (node 0's own token where it has no page, -1 without
 *              nodes): the next tree's node 0
 *   seq_hot    [batch] seq_held + accepted; may be seq_held
 *   path       [num_tokens] in the sequence's rows the kept nodes in order, then -1
 *   history    [batch][history_stride] the kept tokens behind the history_count that were there, and
 *              history_count_out; history_count_out may be history_count (all three NULL: none); past the
 *              stride they are left out and "sequence length" is set
 * and, for each of `layers` layers, K and V row of the j-th kept node to row slots[j-th row of the
 * sequence] of the pool.  A slot past hot_blocks pages is left out and sets "hot block ref", another negative
 * one is left out.  A tree of more than AW_MAX_NODES nodes sets "sequence length", its later nodes are
 * not kept. */
typedef struct aw_accept_desc {
    uint32_t batch, num_tokens;          /* batch <= 2^20, num_tokens <= 2^24 */
    uint32_t layers, kv_heads, head_dim; /* layers 0: no rows are moved; <= 65535 */
    uint32_t history_stride;
    uint64_t hot_blocks;
    uint64_t k_stride, v_stride;         /* elements from node to node, 0 for kv_heads * head_dim */
    uint64_t k_layer_stride, v_layer_stride; /* from layer to layer, 0 for num_tokens * stride */
    uint64_t hot_layer_stride;           /* of the pools, 0 for hot_blocks * 16 * kv_heads * head_dim */
    const int32_t*  parents;             /* [num_tokens] */
    const uint32_t* node_tokens;
    const uint32_t* targets;             /* [num_tokens]: best of aw_ops_adjust_logits, or sampled */
    const uint32_t* token_offsets;
    const uint32_t* seq_held;
    const int64_t*  slots;               /* [num_tokens], of aw_ops_page_tables; may be NULL without layers */
    const uint16_t* k;                   /* [layers][num_tokens][kv_heads][head_dim] */
    const uint16_t* v;                   /* likewise, NULL with hot_v */
    uint16_t* hot_k;                     /* [layers][hot_blocks][16][kv_heads][head_dim] */
    uint16_t* hot_v;
    uint32_t* accepted;
    int32_t*  next_token;
    uint32_t* seq_hot;
    int32_t*  path;
    uint32_t* history;
    const uint32_t* history_count;
    uint32_t* history_count_out;
} aw_accept_desc;

int aw_ops_accept_tree(aw_engine* engine, const aw_accept_desc* desc, void* hip_stream);

/* The host checks of the calls above, as aw_ops_check_rotary. */
int aw_ops_check_tables(const aw_tables_desc* desc, char* msg, size_t msg_len);
int aw_ops_check_logits(const aw_logits_desc* desc, char* msg, size_t msg_len);
int aw_ops_check_accept(const aw_accept_desc* desc, char* msg, size_t msg_len);

/* sizeof(aw_tables_desc), sizeof(aw_logits_desc), sizeof(aw_accept_desc), for bindings. */
void aw_abi_step_desc_sizes(size_t sizes[3]);

/* The tile that a call's product (matmul_qkv: 3, of n[0 .. products) weight rows)
 * of m > 64 rows with 16-byte aligned rows takes on a GPU of `compute_units`, for
 * testing: {activation rows, weight rows, LDS buffers of 64 k}.  Host only.
 * AW_E_UNSUPPORTED where such a product takes none (k % 8 != 0, k > 2 Mi). */
int aw_debug_product_tile(uint32_t compute_units, uint32_t m, const uint32_t* n, uint32_t products, uint32_t k,
                          uint32_t tile[3]);

#ifdef __cplusplus
}
#endif

#endif /* AETHER_OPS_H */
