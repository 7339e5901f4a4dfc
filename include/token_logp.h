/*
 * libtoken_logp_hip.so -- log-probabilities of given tokens, forward and
 * backward, for MI355X (gfx950).
 *
 *   m[r]    = max_v logits[r, v]
 *   S[r]    = sum_v exp((logits[r, v] - m[r]) / temperature)
 *   logp[r] = (logits[r, labels[r]] - m[r]) / temperature - log S[r]
 *   dlogits[r, v] = gout * dlogp[r] / temperature
 *                   * ([v == labels[r]] - exp((logits[r, v] - m[r]) / temperature) / S[r])
 *
 * logits: B x S rows of V elements, element (b, s, v) at b * batch_stride +
 * s * row_stride + v (in elements), of float32, bfloat16 or float16 (dtype 0,
 * 1, 2), aligned to an element.  Everything per row is dense [B, S]: labels
 * int64, logp, dlogp float32, stats two float32 (m, S).  dlogits is dense
 * [B, S, V] of the type of the logits and must not overlap them.
 *
 * A row whose label is `ignore_index` has logp 0 and a gradient of zeros, and
 * its logits are not read; so has the gradient of a row with dlogp 0.  Any
 * other label outside [0, V) makes the row's answers NaN, as does a row of
 * -inf (its probabilities are 0 / 0).
 *
 * Device arrays owned by the caller; the library allocates nothing, keeps no
 * state, never synchronises and launches on `stream`.  Arguments are validated
 * before any HIP call (NL2K_* codes, message from token_logp_last_error()).
 * All results are bitwise repeatable.
 */
#ifndef NL2K_TOKEN_LOGP_H
#define NL2K_TOKEN_LOGP_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* logp, and the rows' stats where a backward follows (NULL otherwise). */
int token_logp_forward(const void* logits, int dtype, const int64_t* labels, float* logp,
                       float* stats, int64_t B, int64_t S, int64_t V, int64_t batch_stride,
                       int64_t row_stride, int64_t ignore_index, float temperature,
                       hipStream_t stream);

/* dlogits from the forward's stats and the gradient of logp; gout [1] scales
 * it where it is not NULL. */
int token_logp_backward(const void* logits, int dtype, const int64_t* labels, const float* stats,
                        const float* dlogp, const float* gout, void* dlogits, int64_t B,
                        int64_t S, int64_t V, int64_t batch_stride, int64_t row_stride,
                        int64_t ignore_index, float temperature, hipStream_t stream);

const char* token_logp_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_TOKEN_LOGP_H */
