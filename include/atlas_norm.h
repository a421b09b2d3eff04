/*
 * atlas_norm.h -- C ABI of layer norm, forward and backward, optionally fused with the
 * residual add in front of it.
 *
 *     h = x + residual            (rounded to act_dtype; h = x without a residual)
 *     y = (h - mean(h)) * rstd(h) * weight + bias,   rstd = 1 / sqrt(var(h) + eps)
 *
 * over vectors of N channels.  The weights may differ from group to group: the input is
 * rows x G vectors (rows, G, N), and vector (r, g) uses weight[g], bias[g].  G = 1 is the
 * usual layer norm; G = heads normalises each head of a (B, T, H, D) activation with a
 * (H, D) weight of its own (the shape of the reference's ln_gamma parameter,
 * atlas_jax/memory_layer.py).
 *
 * Layout: x, residual, y, h, dy, dh, dx are (rows, G, N) contiguous in act_dtype; weight,
 * bias, dweight, dbias (G, N) float32; stats (rows, G, 2) float32, 8-byte aligned: mean
 * and rstd (up to 8 channels: rstd as two floats whose sum it is).
 * Arithmetic is float32 (float64 for vectors of up to 8 channels, whose gradients cancel);
 * outputs in act_dtype are rounded once.  The variance is the mean of the squared differences
 * from the mean (two passes over registers).  Where the mean is above four deviations the forward
 * sums the differences once more and corrects it, so a large mean costs y no digits; stats hold it
 * rounded to float32 (2^-24 of it), which the backward's (h - mean) rstd then contains.  The
 * parameter gradients are summed in a fixed order (no atomics).
 *
 * Conventions (status codes, thread-local error string, stream as void*, caller-owned
 * device buffers) are those of atlas_scan.h.
 */
#ifndef ATLAS_NORM_H_
#define ATLAS_NORM_H_

#include <stddef.h>
#include <stdint.h>

#include "atlas_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  int32_t abi_version; /* ATLAS_ABI_VERSION */
  int32_t act_dtype;   /* ATLAS_F32 or ATLAS_BF16 */
  int64_t rows;        /* >= 0 */
  int32_t G, N;        /* 1 <= G * N <= 2^20 */
  float eps;           /* >= 0 */
  int32_t reserved;    /* 0 */
} AtlasNormParams;

/* Bytes of workspace atlas_layernorm_bwd needs (0 on invalid params, with the message set). */
size_t atlas_layernorm_workspace_bytes(const AtlasNormParams* p);

/* Forward.  residual, weight, bias and stats may be NULL (no residual, ones, zeros, not
 * wanted); h is written when residual is given and may then not be NULL (it may be the
 * buffer of x or of residual). */
int atlas_layernorm_fwd(const AtlasNormParams* p, const void* x, const void* residual, const float* weight,
                        const float* bias, void* y, void* h, float* stats, void* stream);

/* VJP.  h and stats are the forward's (h = x without a residual).  dh (may be NULL): cotangent
 * of h itself, added to dx, which is the cotangent of x and of residual alike (dx may be the
 * buffer of dy or dh).  dweight and dbias may be NULL. */
int atlas_layernorm_bwd(const AtlasNormParams* p, const void* dy, const void* h, const float* weight,
                        const float* stats, const void* dh, void* dx, float* dweight, float* dbias,
                        void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATLAS_NORM_H_ */
