/*
 * libnewton_schulz_hip.so -- orthogonalised updates by Newton-Schulz products,
 * for MI355X (gfx950).
 *
 *   X_0     = U / (||U||_F + eps)          U [m, n]; of its transpose if m > n
 *   A       = X X'
 *   X_(i+1) = a X + (b A + c A A) X        `steps` times
 *   O       = X_steps
 *
 * so that O has U's singular vectors and each singular value s of X_0 in place
 * of p(p(...p(s))), p(s) = a s + b s^3 + c s^5.  newton_schulz writes O;
 * muon_update takes U from a momentum and updates weights with it:
 *
 *   M = mu M + G
 *   U = G + mu M (nesterov) or M
 *   W = (1 - lr weight_decay) W - lr scale O
 *
 * `count` matrices of one shape and type, given by arrays of device pointers
 * (host arrays); matrix element (i, j) at i * row_stride + j, elements of
 * float32, bfloat16 or float16 (dtype 0, 1, 2), aligned to an element.
 *
 * precision 1 (half): X, A and b A + c A A are held in float16, 11 bits each.
 * precision 2 (full): in two float16, 22 bits, three products in place of one.
 * Products are summed in 32 bits, the norm in 64.  Where the
 * shorter side is at most 64 and |a|^(2 steps) <= 1e9, all of it is computed in
 * 64 bits and rounded once, at either precision.  The other operands are
 * scaled by powers of two so that their largest possible values fill float16's
 * range; coefficients under which some singular value in [0, 1] leaves [-4, 4]
 * are refused.  A matrix of zeros gives zeros; one with a NaN or an infinity
 * gives NaN.
 *
 * Device arrays owned by the caller; the library allocates nothing, keeps no
 * state, never synchronises and launches on `stream`.  Arguments are validated
 * before any HIP call (NL2K_* codes, message from newton_schulz_last_error()).
 * Results are bitwise repeatable.  The workspace is scratch without initial
 * contents.
 */
#ifndef NL2K_NEWTON_SCHULZ_H
#define NL2K_NEWTON_SCHULZ_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Scratch bytes for `count` matrices [m, n] (256-byte aligned pointer); 0 for
 * invalid sizes. */
size_t newton_schulz_workspace_bytes(int64_t m, int64_t n, int64_t count, int precision);

/* O of every matrix in `in`, written to `out` in its own type; in-place is
 * allowed. */
int newton_schulz(const void* const* in, int in_dtype, int64_t in_row_stride, void* const* out,
                  int out_dtype, int64_t out_row_stride, int64_t m, int64_t n, int64_t count,
                  int steps, float a, float b, float c, float eps, int precision, void* workspace,
                  size_t workspace_bytes, hipStream_t stream);

/* One step of every weight: updates the momenta and the weights in place.  None
 * of them may overlap another, nor a gradient (but for that of the same weight). */
int muon_update(void* const* weights, int weight_dtype, int64_t weight_row_stride,
                const void* const* grads, int grad_dtype, int64_t grad_row_stride,
                void* const* momenta, int momentum_dtype, int64_t momentum_row_stride, int64_t m,
                int64_t n, int64_t count, float mu, int nesterov, float lr, float weight_decay,
                float scale, int steps, float a, float b, float c, float eps, int precision,
                void* workspace, size_t workspace_bytes, hipStream_t stream);

const char* newton_schulz_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_NEWTON_SCHULZ_H */
