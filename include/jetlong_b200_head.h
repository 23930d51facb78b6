/*
 * jetlong_b200 — C ABI of the vocabulary-head operators: softmax statistics of hidden @ weight^T over a large
 * vocabulary, the cross-entropy loss and its gradients, without the (rows, vocab) logits in memory.  Conventions
 * (status codes, strides in elements, caller-owned memory, explicit stream, nothing synchronises or allocates) are
 * those of jetlong_b200.h.
 */
#ifndef JETLONG_B200_HEAD_H_
#define JETLONG_B200_HEAD_H_

#include "jetlong_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------
 * jl_head_scores — z = hidden weight^T (fp32), per row:
 *   lse = log sum_v e^{z_v},  nll = lse - z_label (0 where label == ignore_index),  top = the lowest v with the largest z_v.
 * A label outside [0, vocab) that is not ignore_index gives nll = NaN; nothing is read out of range.
 * hidden (rows, hidden) and weight (vocab, hidden) bf16 with row strides that are multiples of 8, innermost dimension
 * contiguous, 16-byte aligned; hidden size a multiple of 8.  labels (rows,) int64, may be NULL with nll NULL.
 * nll, lse, top, loss_sum, loss_count, loss_mean may each be NULL.  loss_sum = sum of nll, loss_count = number of rows
 * whose label is not ignore_index, loss_mean = their quotient (fp32 scalars, summed in a fixed order).
 * skip_ignored != 0: rows whose label is ignore_index need no lse (theirs is 0) and may be left out of the product; needs
 * labels, top NULL.
 * workspace: jl_head_scores_workspace_bytes, 16-byte aligned, not initialised by the caller.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const void* hidden;
  const void* weight;
  int64_t hidden_stride, weight_stride;
  const int64_t* labels;
  int64_t ignore_index;
  int64_t rows;
  int32_t hidden_size, vocab;
  float* nll;
  float* lse;
  int64_t* top;
  float* loss_sum;
  float* loss_count;
  float* loss_mean;
  int32_t skip_ignored, reserved;
  void* workspace;
  size_t workspace_bytes;
} jl_head_scores_args;

size_t jl_head_scores_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab, int32_t skip_ignored);
int jl_head_scores(const jl_head_scores_args* args, void* cuda_stream);

/* ---------------------------------------------------------------------------------------------
 * jl_head_grads — gradients of sum_i g_i nll_i, from the lse and nll that jl_head_scores returned for the same operands:
 *   dz_iv = g_i (e^{z_iv - lse_i} - [v == label_i])  (0 where label_i == ignore_index, whatever row i holds),
 *   d_hidden = dz weight,  d_weight = dz^T hidden;
 *   g_i = grad[i] (grad_stride 1) or *grad / (*grad_count if grad_count != NULL; 0 for a count of 0) for every row.
 * z is formed again piece by piece of the vocabulary; a piece of dz is held in bf16 in the workspace, both products
 * accumulate in fp32.  At the label dz_i is g_i (e^{-nll_i} - 1), which does not cancel where the label is all but certain.  d_hidden (rows, hidden) and d_weight (vocab, hidden) bf16 contiguous; either may be NULL.
 * Results do not depend on the timing of anything (no atomics).
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const void* hidden;
  const void* weight;
  int64_t hidden_stride, weight_stride;
  const int64_t* labels;
  int64_t ignore_index;
  int64_t rows;
  int32_t hidden_size, vocab;
  const float* lse;
  const float* nll;
  const float* grad;
  int64_t grad_stride;      /* 0: one scalar for every row, 1: one value per row */
  const float* grad_count;  /* may be NULL; only with grad_stride 0 */
  void* d_hidden;
  void* d_weight;
  void* workspace;
  size_t workspace_bytes;
} jl_head_grads_args;

size_t jl_head_grads_workspace_bytes(int64_t rows, int32_t hidden_size, int32_t vocab);
int jl_head_grads(const jl_head_grads_args* args, void* cuda_stream);

/* Diagnostic (synchronises the device): non-zero if a bounded wait (1 s) inside a head kernel has given up on the current
 * device since the last call; reading a raised status clears it.  The results since the last call are then invalid. */
int jl_head_status(void);

#ifdef __cplusplus
}
#endif
#endif /* JETLONG_B200_HEAD_H_ */
