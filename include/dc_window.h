/*
 * dc_window.h — C ABI of attention with a sliding window and sinks (libdcattn.so, beside dc_attn.h).
 *
 * No counterpart in the reference, whose attention takes such a pattern as a dense (L, S) mask.
 *
 * The query in row l stands at position p = offset + l; key s stands at position s and is visible iff
 *     s <= p  and  (s > p - window  or  s < sinks),
 * the last `window` keys up to the query's own and the first `sinks` ones.  Keys that are not visible
 * are not part of the result, whatever they hold (NaN included), and the work is that of the visible
 * pairs.  A query that sees no key gives out = 0, lse = 0 and zero gradients.
 *
 *   q, grad_out : (B, H, L, E); k, v: (B, Hkv, S, E), H % Hkv == 0 (grouped heads); read through element
 *                 strides of the batch, head and row dims, unit stride along the head dim
 *   out, dq     : contiguous (B, H, L, E); dk, dv: contiguous (B, Hkv, S, E); lse: (B, H, L) float32,
 *                 natural log
 *   scale       : has_scale ? (float)scale (finite) : 1 / sqrt(E)
 *
 * Softmax statistics, sums and products' accumulators are float32, results are rounded once to dtype and
 * are identical from run to run (no atomics).  Device pointers; calls are asynchronous on `stream` (a
 * hipStream_t), launch kernels only and can be captured into HIP graphs.  Workspaces are 256-byte aligned
 * and sized by the *_workspace_size calls for the device current at the call.
 */
#ifndef DC_WINDOW_H
#define DC_WINDOW_H

#include <stddef.h>
#include <stdint.h>

#include "dc_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int64_t batch, heads, kv_heads, q_len, kv_len, head_dim;
    int64_t offset, window, sinks; /* offset, sinks >= 0, window >= 1 */
    int32_t dtype, has_scale;
    double scale;
    int64_t q_stride[3], k_stride[3], v_stride[3]; /* batch, head, row; elements */
    int64_t grad_out_stride[3];                    /* backward */
} dc_window_desc;

/* Largest head_dim of dc_window_fwd and dc_window_bwd, and of dc_window_decode. */
#define DC_WINDOW_MAX_HEAD_DIM 128
#define DC_WINDOW_DECODE_MAX_HEAD_DIM 256

/* (out, lse).  `rest` is optional and used for bfloat16: a tensor like out that takes what rounding out
 * left, itself rounded.  dc_window_bwd forms rowsum(grad_out * out) from both; from the rounded out alone
 * that sum is off by 2^-9 of its terms, which is most of dq where a query sees one key or nearly
 * attends to one.  The workspace is optional: it holds the partial results of key ranges that few rows are
 * split into. */
size_t dc_window_fwd_workspace_size(const dc_window_desc *d);
dc_status dc_window_fwd(const dc_window_desc *d, const void *q, const void *k, const void *v, void *out,
                        void *rest, float *lse, void *workspace, size_t workspace_bytes, void *stream);

/* (dq, dk, dv) from the saved out, rest (or NULL) and lse.  The workspace is required. */
size_t dc_window_bwd_workspace_size(const dc_window_desc *d);
dc_status dc_window_bwd(const dc_window_desc *d, const void *grad_out, const void *q, const void *k,
                        const void *v, const void *out, const void *rest, const float *lse, void *dq, void *dk, void *dv,
                        void *workspace, size_t workspace_bytes, void *stream);

/* One query per sequence (q_len == 1; offset is not used) over a cache of kv_len rows of which sequence
 * b holds lengths[b] (int32 or int64, clamped to 0 .. kv_len; NULL, length_bytes 0: kv_len): the query
 * stands at position lengths[b] - 1.  Rows from lengths[b] on are not read.  The workspace is required. */
size_t dc_window_decode_workspace_size(const dc_window_desc *d);
dc_status dc_window_decode(const dc_window_desc *d, const void *q, const void *k, const void *v,
                           const void *lengths, int32_t length_bytes, void *out, float *lse, void *workspace,
                           size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* DC_WINDOW_H */
