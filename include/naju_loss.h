/*
 * naju_loss.h -- C ABI of the MI355X (gfx950) cross-entropy of the Naju LM
 * training step: the reference's
 *
 *   loss = nn.functional.cross_entropy(logits.reshape(-1, V), y.reshape(-1))
 *
 * under bf16 autocast (/root/reference/evals/lm/train.py:70-74), which
 * evaluates it in float32 on the upcast logits with the defaults
 * ignore_index = -100 and reduction = "mean":
 *
 *   loss = sum_{r valid} ( logsumexp_c x[r,c] - x[r, target[r]] ) / #valid,
 *   valid = target[r] != ignore_index.
 *
 * Layouts: x (logits) [n_rows, n_cols] with x_ld >= n_cols elements between
 * rows, dtype F32, BF16 or F16 (codes of naju_scan.h); target [n_rows] int64;
 * lse [n_rows] float32; loss and scale one float32 each: the mean loss and
 * 1 / #valid (the scale of every valid row's gradient). Arithmetic is
 * float32, the final mean is summed in float64 in a fixed order, so both
 * calls are deterministic. A target outside [0, n_cols) that is not
 * ignore_index gives that row a NaN loss (and NaN gradients) instead of a
 * device fault; no valid row gives a NaN loss, as torch does.
 *
 * Every call is asynchronous on `stream`, allocates nothing and never
 * synchronises the host; errors are reported as in naju_scan.h, with the
 * message in naju_loss_last_error().
 */
#ifndef NAJU_LOSS_H
#define NAJU_LOSS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Message of the last failed call of this thread ("" after a success). */
const char* naju_loss_last_error(void);

/* Bytes of workspace naju_xent_fwd needs (per-row losses); no zero-fill. */
size_t naju_xent_workspace_bytes(int64_t n_rows);

/* Forward: lse[r] = logsumexp of row r, loss and scale as above. One pass over the
 * logits. Replaces the float32 upcast, log_softmax and nll_loss forward that
 * cross_entropy runs under autocast (evals/lm/train.py:74). */
int naju_xent_fwd(const void* x, int64_t x_ld, const int64_t* target, int64_t n_rows, int64_t n_cols, int x_dtype,
                  int64_t ignore_index, float* lse, float* loss, float* scale, void* workspace,
                  size_t workspace_bytes, void* stream);

/* Backward: dx[r,c] = dloss[0] * scale[0] * (exp(x[r,c] - lse[r]) - [c == target[r]])
 * for valid rows, 0 for ignored rows; dx [n_rows, n_cols] with dx_ld >= n_cols,
 * in dx_dtype. dloss is the device float32 gradient of the loss. One pass over
 * the logits; the autograd of the same cross_entropy call, including the cast
 * of the gradient back to the logits' dtype. */
int naju_xent_bwd(const void* x, int64_t x_ld, const int64_t* target, int64_t n_rows, int64_t n_cols, int x_dtype,
                  int64_t ignore_index, const float* lse, const float* scale, const float* dloss, void* dx,
                  int64_t dx_ld, int dx_dtype, void* stream);

/* Forward and gradient in one pass over the logits, for a caller that will
 * take the gradient (autograd's loss.backward()): naju_xent_fwd's outputs,
 * and dx written as naju_xent_bwd writes it for dloss = 1. Each row is read
 * twice by its workgroup (the second time mostly from the caches) instead of
 * a second full pass in the backward. No reference counterpart (the
 * reference's loss is torch's, forward then backward). */
int naju_xent_fwd_grad(const void* x, int64_t x_ld, const int64_t* target, int64_t n_rows, int64_t n_cols,
                       int x_dtype, int64_t ignore_index, float* lse, float* loss, float* scale, void* dx,
                       int64_t dx_ld, int dx_dtype, void* workspace, size_t workspace_bytes, void* stream);

/* The backward after naju_xent_fwd_grad: when dloss[0] is 1 the dx that call
 * wrote is the gradient and nothing is done (each workgroup reads dloss and
 * returns); otherwise dx is rewritten as naju_xent_bwd writes it. */
int naju_xent_bwd_if_scaled(const void* x, int64_t x_ld, const int64_t* target, int64_t n_rows, int64_t n_cols,
                            int x_dtype, int64_t ignore_index, const float* lse, const float* scale,
                            const float* dloss, void* dx, int64_t dx_ld, int dx_dtype, void* stream);

/* The head and its loss in one, without the logits: l = x w^T,
 *   lse[r] = logsumexp_c l[r,c],  row_loss[r] = lse[r] - l[r, target[r]],
 * row_loss 0 for rows whose target is ignore_index, and NaN for a target
 * outside [0, n_cols) otherwise. x [n_rows, d] (x_ld elements between rows)
 * and w [n_cols, d] (w_ld) in `dtype`, BF16 or F16, products summed in
 * float32; the operands' alignment is naju_gated_fwd's (naju_mixer.h); n_rows
 * at most 2^25, n_cols 2^29, d and the strides 2^21. loss and scale (nullable,
 * together): mean != 0 the sum of row_loss over the valid rows times 1 / #valid
 * (NaN without one) and that factor, mean = 0 the sum and 1. Deterministic.
 * Replaces the head's product followed by naju_xent_fwd
 * (evals/lm/train.py:70-74, naju/lm.py:32-33); the workspace
 * holds 8 bytes a row for each 256, 128 or (few rows) 32 columns in place of
 * the logits. */
int naju_linear_xent_fwd(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const int64_t* target,
                         int64_t n_rows, int64_t d, int64_t n_cols, int dtype, int64_t ignore_index, float* lse,
                         float* row_loss, int mean, float* loss, float* scale, void* workspace, size_t workspace_bytes,
                         void* stream);

/* Bytes of workspace (256-byte aligned, no zero-fill) of the forward, or of
 * the backward when backward != 0. That holds
 *   the 16-bit gradient of a piece of the vocabulary's logits: 1 GiB at most, or
 *     512 bytes a row where that is more (above 2^21 rows: a piece has 256
 *     columns at least);
 *   x with the rows of ignored targets zero: 2 bytes for each of n_rows * d (d
 *     rounded up to 8), and 4 bytes a row;
 *   where the vocabulary takes several pieces, dx in float32: 4 n_rows d bytes;
 *   the float32 parts of a product split over k, of one product at a time (none
 *     where its result has many tiles): for d of 256 and more at most ten times,
 *     below 64 times, the larger of dx and a piece's dw in float32. */
size_t naju_linear_xent_workspace_bytes(int64_t n_rows, int64_t d, int64_t n_cols, int backward);

/* Backward of naju_linear_xent_fwd, the logits formed again by pieces of the
 * vocabulary: dx [n_rows, d] in `dtype` and dw [n_cols, d] in dw_dtype
 * (`dtype` or F32), contiguous, each nullable. The gradient of row r's loss
 * is dloss[r * dloss_step] * scale[0] (dloss_step 0: one value for all rows;
 * scale nullable: 1), device float32. Deterministic. n_rows = 0 writes
 * nothing. */
int naju_linear_xent_bwd(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const int64_t* target,
                         int64_t n_rows, int64_t d, int64_t n_cols, int dtype, int64_t ignore_index, const float* lse,
                         const float* scale, const float* dloss, int64_t dloss_step, void* dx, void* dw, int dw_dtype,
                         void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NAJU_LOSS_H */
