/*
 * atlas_decay.h -- C ABI of decay attention: causal linear attention whose state decays
 * by a factor of its own in each head.
 *
 * For every batch b and head h, with l = exp(log_decay[h]):
 *
 *     S_t = l S_{t-1} + k_t v_t^T          (D x D, row = key channel, column = value channel)
 *     y_t = scale * q_t^T S_t
 *
 * It is the memory M_t = alpha M_{t-1} + ... of the linear scan (atlas_scan.h) without its
 * error term, Omega window, momentum and Polar Express, so a whole chunk is a few dense
 * products.  atlas_decay_fwd / _bwd take whole sequences (prompts, training);
 * atlas_decay_step advances a pool of states by one or a few tokens (generation).
 *
 * Layout
 *  - q, k, v: (B, T, H, D) in act_dtype, D channels contiguous, any strides between
 *    batches, tokens and heads (in elements; views of a fused projection need no copy,
 *    broadcast axes have stride 0).  y, dy, dq, dk, dv: (B, T, H, D) contiguous, act_dtype.
 *  - log_decay, dlog_decay: (H) float32.  log_decay <= 0 in use; 0 never forgets, -infinity
 *    keeps only the current token.
 *  - states: (B, H, D, D) float32 contiguous.
 *  - 1 <= D <= 128.  T = 0 is a valid call (the states pass through).
 *
 * Arithmetic: sums, decays and states are float32.  bf16 activations with D a multiple of
 * 8 and 16-byte aligned rows run on the tcgen05 tensor cores; other calls run in float32
 * on the CUDA cores.  On the tensor cores what reaches float32 outputs (states, dlog_decay) is
 * kept to float32 accuracy by splitting float32 operands into three bf16 parts; for the bf16
 * outputs operands are rounded to fewer bits: the decayed scores of a chunk to bf16 (q k^T
 * before its products with v and dy, dy v^T before its products with k and q), the state in
 * q S and the cotangent state in k R (for dv) to two bf16 parts, 16 bits.  The relative error of y, dq,
 * dk and dv is then about 1.8e-3, where the one rounding to bf16 alone leaves 1.66e-3; the rounded
 * scores make nearly all of the difference.
 * Causality holds for finite inputs; an infinity or NaN in v or k of a token reaches the
 * outputs of its own 64-token chunk as well as those after it, an infinity mostly as NaN.
 *
 * Conventions (status codes, thread-local error string, stream as void*, caller-owned
 * device buffers) are those of atlas_scan.h.
 */
#ifndef ATLAS_DECAY_H_
#define ATLAS_DECAY_H_

#include <stddef.h>
#include <stdint.h>

#include "atlas_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  int32_t abi_version; /* ATLAS_ABI_VERSION */
  int32_t B, T, H, D;
  int32_t act_dtype; /* ATLAS_F32 or ATLAS_BF16 */
  float scale;       /* of the read-out */
  int32_t aligned16; /* 1: every buffer of the calls is 16-byte aligned (then checked); what the
                      * tensor cores need, beside bf16, D % 8 == 0 and strides of the axes longer
                      * than 1 that are positive multiples of 8 */
  /* elements between batches, tokens and heads of q, k and v */
  int64_t q_stride[3], k_stride[3], v_stride[3];
} AtlasDecayParams;

/* Bytes of the forward's `saved` buffer: the state entering every 64-token chunk
 * (0 on invalid params, with the message set, and for empty problems). */
size_t atlas_decay_saved_bytes(const AtlasDecayParams* p);

/* Bytes of workspace of a forward without `saved`, of one with it, and of the backward (0 on invalid params,
 * and where none is needed). */
size_t atlas_decay_fwd_workspace_bytes(const AtlasDecayParams* p);
size_t atlas_decay_saved_workspace_bytes(const AtlasDecayParams* p);
size_t atlas_decay_bwd_workspace_bytes(const AtlasDecayParams* p);

/* Forward.  state_in may be NULL (zeros); state_out = S after token T - 1 and may be the same
 * buffer as state_in; saved may be NULL when no backward follows. */
int atlas_decay_fwd(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                    const float* log_decay, const float* state_in, void* y, float* state_out, void* saved,
                    void* workspace, size_t workspace_bytes, void* stream);

/* VJP of atlas_decay_fwd.  saved: the forward's, same params.  dstate_out: cotangent of
 * state_out or NULL (zeros).  dstate_in (cotangent of state_in) and dlog_decay may be NULL.
 * All outputs are overwritten; results do not depend on timing (no atomics). */
int atlas_decay_bwd(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                    const float* log_decay, const void* saved, const void* dy, const float* dstate_out, void* dq,
                    void* dk, void* dv, float* dlog_decay, float* dstate_in, void* workspace,
                    size_t workspace_bytes, void* stream);

/* The recurrent form: token by token from state_in to state_out (which may be the same
 * buffer).  The decay is applied as a float pair, so that states kept over thousands of tokens stay
 * as near to float64 as those of atlas_decay_fwd.  slots NULL: the states are (B, H, D, D) and sequence b uses row b.  Otherwise
 * they are pools of n_slots rows (n_slots, H, D, D) and sequence b uses row slots[b] (int32);
 * the running sequences' slots differ from one another, and a slot outside [0, n_slots)
 * marks an idle sequence: its y is 0 and no state is touched.  Rows that no sequence names
 * are left as they are. */
int atlas_decay_step(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                     const float* log_decay, const float* state_in, const int32_t* slots, int32_t n_slots, void* y,
                     float* state_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATLAS_DECAY_H_ */
