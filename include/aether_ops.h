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
