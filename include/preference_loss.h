/*
 * libpreference_loss_hip.so -- preference loss of paired log ratios, from
 * logits, for MI355X (gfx950).
 *
 *   logp[r]  = log-probability of row r's label (token_logp.h), 0 where ignored
 *   seq[i]   = sum of logp over sequence i, divided by the number of its
 *              labels that count (at least 1) where `average` is set
 *   h[i]     = beta (seq[i] - ref_seq[i])
 *   delta[i] = h[i] - h[i + N]            sequence i chosen, i + N rejected, i < N
 *   loss     = 1/N sum_i ((1 - eps) softplus(-delta[i]) + eps softplus(delta[i]))
 *   coef     = d loss / d logp
 *            = +- beta / N (eps sigmoid(delta) - (1 - eps) sigmoid(-delta)) [/ count]
 *   dlogits  = coef (onehot(label) - softmax)
 *
 * eps is `label_smoothing`.  logits as in token_logp.h.  Without cu_seqlens the
 * 2 N sequences are the batch entries, B = 2 N; with it the rows of B = 1 hold
 * them one after the other, sequence i from cu_seqlens[i] to cu_seqlens[i + 1]
 * (int64, 2 N + 1 of them, on the device; not validated: rows in no sequence
 * get zeros, offsets are clamped into the rows).  N is at most 2^24 - 1.
 * ref_seq [2 N] (NULL: zeros) and seq_logp [2 N] float32.
 *
 * Sums over tokens and pairs are taken in 64 bits in a fixed order: all
 * results are bitwise repeatable.  Workspace: scratch without initial
 * contents.  The other conventions are those of token_logp.h.
 */
#ifndef NL2K_PREFERENCE_LOSS_H
#define NL2K_PREFERENCE_LOSS_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Scratch bytes of the forward (8-byte aligned) for B * S rows and `pairs`
 * pairs; 0 for invalid sizes. */
size_t preference_loss_workspace_bytes(int64_t B, int64_t S, int64_t pairs);

/* loss [1], seq_logp [2 N], and for a backward stats [B, S, 2] and coef [B, S]
 * (both or neither NULL). */
int preference_loss_forward(const void* logits, int dtype, const int64_t* labels,
                            const float* ref_seq, const int64_t* cu_seqlens, int64_t pairs,
                            float* loss, float* seq_logp, float* stats, float* coef, int64_t B,
                            int64_t S, int64_t V, int64_t batch_stride, int64_t row_stride,
                            int64_t ignore_index, float beta, float label_smoothing, int average,
                            void* workspace, size_t workspace_bytes, hipStream_t stream);

/* dlogits of the forward's loss times gout [1] (a device pointer, or NULL for 1). */
int preference_loss_backward(const void* logits, int dtype, const int64_t* labels,
                             const float* stats, const float* coef, const float* gout,
                             void* dlogits, int64_t B, int64_t S, int64_t V, int64_t batch_stride,
                             int64_t row_stride, int64_t ignore_index, hipStream_t stream);

const char* preference_loss_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_PREFERENCE_LOSS_H */
