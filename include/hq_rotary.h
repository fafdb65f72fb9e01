/*
 * hq_rotary.h — C ABI of the query and key heads' way from the projections to the attention (gfx950).
 *
 * What an attention layer does between its q | k | v projections (include/hq_qgemm.h) and its scores
 * (include/hq_attn.h): a norm of each query and key head, the rotation by the token's position and, for keys and
 * values, the way into the cache's pages. Conventions are those of hq_qgemm.h and hq_attn.h: device pointers,
 * caller-owned buffers, a call returns after enqueueing its kernel on `stream`, on error nothing is enqueued,
 * results are deterministic.
 *
 * Definition. x is one head of one token, D elements, w the norm's weight, p the token's position:
 *   y = x * w / sqrt(mean(x^2) + eps)                  (no weight: y = x)
 *   a_i = 2 pi p turns[i],  i < R / 2
 *   (u, v) = (y[i], y[i + R / 2])  HQ_ROTARY_HALF,  or  (y[2 i], y[2 i + 1])  HQ_ROTARY_INTERLEAVED
 *   out: scale * (u cos a_i - v sin a_i) in u's place, scale * (v cos a_i + u sin a_i) in v's; y from R on.
 * p turns[i] is kept in 64 bits until whole turns are taken off, everything else in fp32; the output is rounded once.
 */
#ifndef HQ_ROTARY_H
#define HQ_ROTARY_H

#include "hq_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef HQ_ENUM(hq_rotary_layout) { HQ_ROTARY_HALF = 1, HQ_ROTARY_INTERLEAVED = 2 } hq_rotary_layout;

/* How heads are rotated. */
typedef struct hq_rotary {
    const double* turns;     /* [dim / 2]: turns of pair i from one position to the next */
    uint32_t dim;            /* R: a multiple of 16, 16 to head_dim */
    hq_rotary_layout layout;
    float scale;             /* of the rotated part: positive and finite (1: a rotation alone) */
} hq_rotary;

/* Heads of a call: element (t, h, d) of In at t * in_row + h * in_head + d, of Out likewise, no two of Out in one place.
 * Strides are in elements and multiples of 8, In and Out 16-byte aligned. Out may be In with the same strides
 * (in place), else they are apart; q's Out is apart from k's In and Out and from V, k's Out from q's In. weight: fp32 [head_dim],
 * 16-byte aligned, or NULL: no norm. eps: not negative, finite. */
typedef struct hq_rotary_heads {
    const void* In;
    void* Out;
    int64_t in_row, in_head;
    int64_t out_row, out_head;
    const float* weight;
    uint32_t heads;
    float eps;
} hq_rotary_heads;

/* Norm and rotation of q and k (NULL: q alone) of `tokens` tokens at positions[t] (int32). head_dim: 64, 128 or 256. */
hq_status hq_rotate(const hq_rotary* rotary, const hq_rotary_heads* q, const hq_rotary_heads* k, uint32_t tokens,
                    uint32_t head_dim, hq_dtype dtype, const int32_t* positions, hq_stream stream);

/* hq_cache_append with k normed and rotated on its way into the pages (k's Out and its strides are not used), and q
 * (NULL: none) to its Out in the same launch. A token's position is its place in its row, from 0. What hq_cache_append
 * skips and reports is skipped and reported here, q's heads of those tokens are written all the same (of a row out of
 * range as at position 0); tokens of no sequence are left as they are. */
hq_status hq_cache_append_rotated(const hq_kv_cache* cache, uint32_t layer, const hq_rotary* rotary, const hq_rotary_heads* q,
                                  const hq_rotary_heads* k, const void* V, int64_t v_row, int64_t v_head, uint32_t tokens,
                                  const int32_t* rows, const int32_t* cu, uint32_t n, hq_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* HQ_ROTARY_H */
