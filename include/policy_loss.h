/*
 * libpolicy_loss_hip.so -- clipped policy loss with a KL term, from logits,
 * for MI355X (gfx950).
 *
 *   logp   = log-probability of the row's label (token_logp.h)
 *   ratio  = exp(logp - old_logp)
 *   kl     = exp(ref_logp - logp) - (ref_logp - logp) - 1
 *   term   = -min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef kl
 *   loss   = sum_r w[r] term[r] / D
 *   coef   = d loss / d logp
 *          = w / D (-ratio A where the clamp does not hold the minimum, else 0,
 *                   + kl_coef (1 - exp(ref_logp - logp)))
 *   dlogits = coef / temperature (onehot(label) - softmax)
 *
 * w is 0 where the label is `ignore_index`, else the mask's value (1 without a
 * mask); D is `denom` where that is > 0, else the sum of w.  A row of weight 0
 * counts for nothing whatever it and its other inputs hold: its logits are not
 * read, its logp is 0 and its gradient zeros.  Where every weight is 0 so are
 * the loss and all gradients.  A counted label outside [0, V) makes the loss
 * and the row's gradient NaN.
 *
 * logits as in token_logp.h.  labels, old_logp, ref_logp (NULL: no KL term),
 * mask and logp, coef are dense [B, S]; the advantage of (b, s) is at
 * b * adv_bs + s * adv_ss, so one a sequence has adv_ss = 0.  mask_kind: 0
 * none, 1 bytes (0 or 1), 2 float32 weights.
 *
 * The loss is summed in 64 bits in a fixed order: all results are bitwise
 * repeatable.  Workspace: scratch without initial contents.  The other
 * conventions are those of token_logp.h.
 */
#ifndef NL2K_POLICY_LOSS_H
#define NL2K_POLICY_LOSS_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Scratch bytes of both forward entries (8-byte aligned); 0 for invalid sizes. */
size_t policy_loss_workspace_bytes(int64_t B, int64_t S);

/* loss [1], logp, and for a backward stats [B, S, 2] and coef [B, S] (both or
 * neither NULL). */
int policy_loss_forward(const void* logits, int dtype, const int64_t* labels,
                        const float* old_logp, const float* advantages, int64_t adv_bs,
                        int64_t adv_ss, const float* ref_logp, const void* mask, int mask_kind,
                        float* loss, float* logp, float* stats, float* coef, int64_t B, int64_t S,
                        int64_t V, int64_t batch_stride, int64_t row_stride, int64_t ignore_index,
                        float temperature, float clip_low, float clip_high, float kl_coef,
                        float denom, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* dlogits of the forward's loss times gout [1] (a device pointer, or NULL for 1). */
int policy_loss_backward(const void* logits, int dtype, const int64_t* labels, const float* stats,
                         const float* coef, const float* gout, void* dlogits, int64_t B, int64_t S,
                         int64_t V, int64_t batch_stride, int64_t row_stride,
                         int64_t ignore_index, float temperature, hipStream_t stream);

/* loss, logp and the loss's dlogits, dense [B, S, V], with the logits read
 * once.  dlogits may be the logits themselves where those are dense; it must
 * not overlap them otherwise. */
int policy_loss_and_grad(const void* logits, int dtype, const int64_t* labels,
                         const float* old_logp, const float* advantages, int64_t adv_bs,
                         int64_t adv_ss, const float* ref_logp, const void* mask, int mask_kind,
                         float* loss, float* logp, void* dlogits, int64_t B, int64_t S, int64_t V,
                         int64_t batch_stride, int64_t row_stride, int64_t ignore_index,
                         float temperature, float clip_low, float clip_high, float kl_coef,
                         float denom, void* workspace, size_t workspace_bytes, hipStream_t stream);

const char* policy_loss_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_POLICY_LOSS_H */
