/*
 * dc_rotary.h — C ABI of the position rotation of queries and keys, alone or behind each head's
 * root-mean-square norm, with gradients (libdcattn.so, beside dc_attn.h).
 *
 * No counterpart in the reference, whose attention starts at q and k as they are given.
 *
 * A token at position p turns pair i of a head's first rotary_dim dims by the angle a = p * inv_freq[i]:
 *     y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
 * with the pair (i, i + rotary_dim / 2), or (2i, 2i + 1) when `interleaved`; m is `magnitude`; the
 * other dims are passed on.  With `norm` the rotation takes u = x r w in place of x, where
 * r = 1 / sqrt(mean(x^2) + eps) over the head's dims and w is a weight per dim (NULL: 1).
 * Angles are formed in float64, everything else in float32; results are rounded once to dtype.
 *
 *   q, k         : (B, H, L, E) and (B, Hkv, L, E), read through element strides of the batch, head
 *                  and row dims, unit stride along the head dim (a projection's (B, L, H, E) is other
 *                  strides)
 *   grad_*       : gradients of the outputs, of the same shapes, through strides of their own
 *   q_out, k_out, dq, dk : contiguous (B, H, L, E) / (B, Hkv, L, E)
 *   inv_freq     : rotary_dim / 2 float64 values, radians per position
 *   positions    : int32 or int64, position of (b, l) at b * pos_stride_b + l * pos_stride_l; NULL
 *                  (pos_bytes 0): offset + l
 *   weights, their gradients : contiguous E values of weight_dtype
 *
 * k (with k_out, grad_k, dk) may be left out with kv_heads 0.  Outputs must not overlap inputs.
 * Device pointers; calls are asynchronous on `stream` (a hipStream_t) and launch kernels only.
 */
#ifndef DC_ROTARY_H
#define DC_ROTARY_H

#include <stddef.h>
#include <stdint.h>

#include "dc_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int64_t batch, heads, kv_heads, q_len, head_dim, rotary_dim;
    int32_t dtype, weight_dtype; /* dc_dtype of q, k, outputs and gradients; of the weights */
    int32_t interleaved, norm;   /* 0 / 1 */
    int32_t pos_bytes;           /* 0 (no positions), 4 or 8 */
    int32_t reserved;            /* 0 */
    int64_t offset, pos_stride_b, pos_stride_l;
    double magnitude, eps;
    int64_t q_stride[3], k_stride[3];           /* batch, head, row; elements */
    int64_t grad_q_stride[3], grad_k_stride[3]; /* backward */
} dc_rotary_desc;

/* Largest head_dim of these entry points. */
#define DC_ROTARY_MAX_HEAD_DIM 512

dc_status dc_rotary_fwd(const dc_rotary_desc *d, const void *q, const void *k, const void *q_weight,
                        const void *k_weight, const double *inv_freq, const void *positions, void *q_out,
                        void *k_out, void *stream);

/* Gradients of q, k and, with norm, of the weights that are given (dq_weight, dk_weight of
 * weight_dtype; NULL where not wanted), summed in a fixed order.  Without norm q, k, weights and
 * workspace may be NULL.  The workspace holds the weight gradients' partial sums. */
size_t dc_rotary_bwd_workspace_size(const dc_rotary_desc *d);
dc_status dc_rotary_bwd(const dc_rotary_desc *d, const void *grad_q, const void *grad_k, const void *q,
                        const void *k, const void *q_weight, const void *k_weight, const double *inv_freq,
                        const void *positions, void *dq, void *dk, void *dq_weight, void *dk_weight,
                        void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* DC_ROTARY_H */
