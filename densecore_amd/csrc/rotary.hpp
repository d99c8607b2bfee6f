// Parameter block and launchers of the position rotation (rotary.hip), sizes validated by the ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dc {

// One tensor of rows (batch, heads, q_len) x head_dim: queries or keys.
struct RotRows {
    const void *x;         // inputs (null in the backward without norm)
    const void *g;         // gradients of the outputs (backward)
    void *out;             // contiguous
    const void *w;         // weight per dim, or null
    int64_t xs[3], gs[3];  // strides of x and g: batch, head, row
    int heads;
};

struct RotArgs {
    RotRows t[2];  // queries, keys
    const double *freq;
    const void *pos;
    int pos_bytes;
    int64_t offset, pos_sb, pos_sl;
    int64_t tokens;  // batch * q_len
    int L, E, R;
    float magnitude, eps;
    bool interleaved, norm, w_bf16;
    int hb;              // heads a group of lanes takes one after the other (same angles)
    float *part[2];      // weight gradients' partial sums, (blocks, E) each; null: not wanted
    void *dw[2];
    int nblk[2];         // workgroups of each tensor in the backward with norm
};

// Forward, and the backward without norm (`inverse`: x = g, turned the other way).
hipError_t launch_rotary(const RotArgs &a, bool bf16, bool inverse, hipStream_t st);
hipError_t launch_rotary_norm_bwd(const RotArgs &a, bool bf16, hipStream_t st);
constexpr int kRotMaxBlocks = 1024;  // workgroups per tensor whose partial sums are kept

}  // namespace dc
