/*
 * hq_ssm.h — C ABI of a state space layer's mixer between its projections (gfx950).
 *
 * The short causal convolution and the selective scan behind it, over packed prompts or single tokens, and the
 * states that sequences keep from call to call. Conventions are those of hq_qgemm.h and hq_attn.h: device
 * pointers, caller-owned buffers, streams, workspaces and status codes; a call returns after enqueueing its
 * kernels on `stream`, on error nothing is enqueued, results are deterministic.
 *
 * Sequences. Sequence i of a call is row rows[i] of the states (rows NULL: row i); its new tokens are
 * [cu[i], cu[i + 1]) of the inputs (cu: int32 [n + 1], not falling, values outside 0..tokens are clamped; NULL: token i
 * alone, then tokens = n). held[i] = 0: the sequence begins with this call, its states are taken as zero whatever they
 * hold (held NULL: all continue). A row appears once. A sequence whose row is out of range, or appears before it in the
 * list, is reported (HQ_CACHE_BAD_ROW in *status) and computed from zero states that are not kept; rows whose
 * `refused` word is not zero are computed and not kept, so that a step that the key/value cache had no room for can be run
 * again. Sequences without tokens keep their states. Tokens of no sequence are left as they are.
 *
 * Convolution, W taps over each channel c; x_s of s < 0 are the row's last inputs before the call:
 *   y[t, c] = f(bias[c] + sum_{j < W} w[c, j] x[t - W + 1 + j, c]),   f(u) = u or u / (1 + exp(-u))
 * Scan, head h with its group g = h / (heads / groups); the state S is [head_dim][state_dim]:
 *   dt = dt_raw[t, h] + dt_bias[h], or log(1 + exp(that))
 *   S = exp(A[h] dt) S + dt x[t, h, :] B[t, g, :]^T
 *   y[t, h, :] = S C[t, g, :] + D[h] x[t, h, :],   times z / (1 + exp(-z)) with a gate z
 * States, decays and sums are kept in fp32 (sums of a chunk's exponents in 64 bits); outputs are rounded once. Calls of a few
 * tokens a sequence are computed so throughout. Longer ones go in chunks of tokens as products of 16-bit operands
 * (hq_describe_ssm says which), into which fp32 values enter as two or three parts: a state's terms with 22 bits (fp16: or to 2^-39
 * of the largest term of their channel and chunk), the state with 16 (fp16: 22, or to 2^-39 of its channel's largest), the
 * weights of a chunk's own tokens with 16.
 * Values that are not finite: tokens before one, other sequences, heads (another group's, for B and C) and, for an x or a state,
 * other channels are as without it. What it enters is not finite; whether an infinity or NaN depends on the kernel.
 */
#ifndef HQ_SSM_H
#define HQ_SSM_H

#include "hq_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HQ_SSM_MAX_BATCH 1024u /* sequences of one call */

/* What sequences keep. conv: the last width - 1 inputs, oldest first, of layer l and row r at l * conv_layer + r * conv_row,
 * [width - 1][channels]; ssm: fp32 [heads][head_dim][state_dim] at l * ssm_layer + r * ssm_row. Strides are in elements,
 * multiples of 8 (conv) and 4 (ssm), both 16-byte aligned. Either may be NULL where a call does not use it. */
typedef struct hq_state_cache {
    void* conv;
    float* ssm;
    int64_t conv_layer, conv_row, ssm_layer, ssm_row;
    uint32_t layers, rows;
    uint32_t channels /* a multiple of 8 */, width /* 2 to 4 */;
    uint32_t heads, head_dim /* 64 or 128 */, state_dim /* 64, 128 or 256 */;
    hq_dtype dtype;          /* of the activations and of conv */
    uint32_t* status;        /* one word, to which calls OR HQ_CACHE_* faults (the caller clears it) */
    const int32_t* refused;  /* per row, an hq_kv_cache's, or NULL */
} hq_state_cache;

/* Convolution of tokens rows of X ([tokens][channels], ldx elements apart) to Y. W: fp32 [channels][width], bias: fp32
 * [channels] or NULL, 16-byte aligned; X, Y 16-byte aligned, ldx, ldy multiples of 8. Y is apart from X. */
hq_status hq_ssm_conv(const hq_state_cache* cache, uint32_t layer, const void* X, int64_t ldx, void* Y, int64_t ldy, const float* W,
                      const float* bias, int silu, uint32_t tokens, const int32_t* rows, const int32_t* held, const int32_t* cu,
                      uint32_t n, hq_stream stream);

/* Inputs and outputs of a scan, strides in elements: X, Y, Z (NULL: no gate) [tokens][heads][head_dim], B, C
 * [tokens][groups][state_dim], dt [tokens][heads] with its heads side by side, fp32 (dt_f32) or of the activations' type.
 * X, B, C, Y, Z: 16-byte aligned, strides multiples of 8 (rows at most 2^22, dt's too). A, D (NULL: 0), dt_bias (NULL: 0): fp32 [heads], A not
 * positive. heads: a multiple of groups. Y may be Z with the same strides (in place), else it is apart from all inputs. */
typedef struct hq_ssm_io {
    const void* X;
    const void* B;
    const void* C;
    const void* dt;
    const void* Z;
    void* Y;
    const float* A;
    const float* D;
    const float* dt_bias;
    int64_t x_row, x_head, b_row, b_group, c_row, c_group, dt_row, z_row, z_head, y_row, y_head;
    uint32_t tokens, groups;
    int dt_f32, softplus;
} hq_ssm_io;

/* Workspace of one hq_ssm_scan call on the current device (0: none), as hq_workspace_bytes; cu: whether the call has one.
 * The size does not fall as tokens and max_len grow: one taken at the largest serves every call of as many sequences. */
hq_status hq_ssm_workspace_bytes(uint32_t tokens, uint32_t n, int cu, uint32_t heads, uint32_t groups, uint32_t head_dim,
                                 uint32_t state_dim, uint32_t max_len, size_t* bytes);
/* The kernels that such a call runs and the workspace that it uses, as text. */
hq_status hq_describe_ssm(uint32_t tokens, uint32_t n, int cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim,
                          uint32_t max_len, char* buf, size_t buf_len);
/* Scan. max_len: no sequence has more new tokens (0: tokens); it only chooses how the work is split (several prompts of one
 * length take up to twice as long without it), as does the mean number of tokens, which alone chooses between the kernels:
 * single tokens and a long chunk are faster as two calls. */
hq_status hq_ssm_scan(const hq_state_cache* cache, uint32_t layer, const hq_ssm_io* io, const int32_t* rows, const int32_t* held,
                      const int32_t* cu, uint32_t n, uint32_t max_len, void* workspace, size_t workspace_bytes, hq_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* HQ_SSM_H */
