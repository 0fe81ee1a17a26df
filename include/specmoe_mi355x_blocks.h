/*
 * specmoe_mi355x_blocks.h -- what a mixture-of-experts block needs around the products of
 * specmoe_mi355x_products.h, with gradients: the norm before it, the routing of its tokens, and the
 * rows' way to the experts and back. Same library, same conventions: plain device pointers and sizes,
 * stream-ordered on `stream`, no host synchronisation, no device allocation (scratch is the caller's
 * workspace, 16-byte aligned), status codes of specmoe_mi355x.h. Calls are re-entrant for distinct
 * workspaces; a captured graph keeps using the workspace of its calls. Results of a call do not depend
 * on timing: every sum runs in a fixed order. No counterpart in the reference, which serves only and
 * leaves these operators to its framework.
 *
 * Rows of matrices lie *_stride elements apart (>= their length), elements of a row side by side;
 * results without a stride are dense. Any alignment of elements (16-byte aligned rows are faster).
 * dtype codes are those of specmoe_mi355x.h. Outputs overlap no operand.
 */
#ifndef SPECMOE_MI355X_BLOCKS_H
#define SPECMOE_MI355X_BLOCKS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms ------------------------------------------------------------------------------------- */

enum smx_norm_kind {
  SMX_NORM_LAYER = 0, /* (s - mean(s)) / sqrt(var(s) + eps) */
  SMX_NORM_RMS = 1    /* s / sqrt(mean(s^2) + eps) */
};

/*
 * s = x + residual, rounded to `dtype` and kept in `sum`; or s = x without a residual (sum NULL).
 * y = norm(s) * weight + bias over rows of H <= 16384 columns. weight, bias [H] may be NULL and are of
 * `weight_dtype`: `dtype`, or fp32. stats: NULL, or what smx_norm_grad needs: fp32 [rows] of
 * 1 / sqrt(..) for SMX_NORM_RMS, [rows][2] of mean and 1 / sqrt(..) for SMX_NORM_LAYER.
 */
int smx_norm(int kind, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
             int dtype, int64_t rows, int64_t H, const void* weight, const void* bias, int weight_dtype,
             float eps, void* y, void* sum, float* stats, void* stream);

/* Bytes of workspace of smx_norm_grad for grad_weight and grad_bias; 0 for bad sizes. */
size_t smx_norm_grad_workspace_size(int kind, int64_t rows, int64_t H, int dtype);

/*
 * Gradients for the gradient grad_y of y and, with a residual, grad_sum of the kept sum (or NULL):
 *     g = grad_y * weight, n = norm(s)
 *     grad_x = (g - mean(g) - n mean(g n)) / sqrt(..) + grad_sum        (SMX_NORM_RMS: without mean(g))
 *     grad_weight = the column sums of grad_y n, grad_bias those of grad_y, of `weight_dtype`
 * grad_x is the residual's gradient too. Each may be NULL where it is not wanted. s and stats: those of
 * the forward call.
 */
int smx_norm_grad(int kind, const void* grad_y, int64_t grad_y_stride, const void* grad_sum,
                  int64_t grad_sum_stride, const void* s, int64_t s_stride, int dtype, int64_t rows,
                  int64_t H, const void* weight, int weight_dtype, const float* stats, void* grad_x,
                  void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                  void* stream);

/* ---- routing ----------------------------------------------------------------------------------- */

enum smx_scoring {
  SMX_SCORE_SOFTMAX = 0, /* over all experts */
  SMX_SCORE_SIGMOID = 1
};

/* Bytes of workspace of smx_route; 0 for bad sizes. */
size_t smx_route_workspace_size(int64_t T, int64_t E, int64_t k);

/*
 * The experts of each token, and the picks in the experts' order. logits [T, E] of `dtype`, 1 <= E <=
 * 1024, 1 <= k <= 16, T k < 2^31.
 *   choice  score + bias (fp32 [E]), or without a bias the score
 *   groups  num_groups (<= 64, a divisor of E) groups of consecutive experts, of which the top_groups
 *           best stay: by their best choice, or with a bias by the sum of their two best
 *   picks   the k best experts by choice, in that order; ties go to the lower index everywhere. Choices
 *           are compared as exact scores would be: in 64 bits where 32 cannot tell them apart. NaN comes
 *           first, as the largest. An expert whose logit or choice is -inf is nobody's pick.
 *   weight  the pick's score, divided by the sum of the token's picks' (renormalize), times scale
 * Where a token has fewer than k experts, the picks left over have id -1 and weight 0.
 *
 * weights fp32 [T, k], ids int32 [T, k]. order int32 [T k]: the picks (token k + j) sorted by expert, and
 * by number within an expert; picks of nobody come last, as their complement (~). places int32 [T, k]:
 * where each pick is in that order, the complement for picks of nobody. offsets int64 [E + 1]: expert
 * e's picks are offsets[e] .. offsets[e + 1] - 1 (the group_offsets of smx_grouped_linear). order,
 * places and offsets may be NULL together: then no order is made.
 */
int smx_route(const void* logits, int64_t logits_stride, int dtype, int64_t T, int64_t E, int64_t k,
              int scoring, const float* bias, int64_t num_groups, int64_t top_groups, int renormalize,
              float scale, float* weights, int32_t* ids, int32_t* places, int32_t* order,
              int64_t* offsets, void* workspace, size_t workspace_bytes, void* stream);

/* The gradient of the logits (dense, of `dtype`) for grad_weights fp32 [T, k]; ids of the forward call. */
int smx_route_grad(const float* grad_weights, const void* logits, int64_t logits_stride, int dtype,
                   int64_t T, int64_t E, int64_t k, int scoring, int renormalize, float scale,
                   const int32_t* ids, void* grad_logits, void* stream);

/* ---- rows to the experts and back ---------------------------------------------------------------- */

/*
 * rows [T k, H]: at places[t, j] the row t of x [T, H], or zeros for a pick of nobody (negative: the row at
 * ~places[t, j]). Places outside [0, T k) write nothing. 1 <= k <= 16, T k < 2^31. The gradient of x is
 * smx_combine_rows of the rows' without weights.
 */
int smx_dispatch_rows(const void* x, int64_t x_stride, int dtype, int64_t T, int64_t H,
                      const int32_t* places, int64_t k, void* rows, void* stream);

/*
 * y [T, H]: residual (may be NULL) + the sum over j of weights[t, j] (fp32 [T, k]; NULL: 1) times the row
 * places[t, j] of rows [T k, H]; summed in fp32, rounded once. Picks of nobody and places outside [0, T k)
 * are left out.
 */
int smx_combine_rows(const void* rows, int64_t rows_stride, int dtype, int64_t T, int64_t H,
                     const int32_t* places, int64_t k, const float* weights, const void* residual,
                     int64_t residual_stride, void* y, void* stream);

/*
 * Gradients of smx_combine_rows for grad_y: grad_rows [T k, H] = weights[t, j] grad_y[t] at places[t, j]
 * (zeros at rows of picks of nobody), grad_weights fp32 [T, k] = the product of that row and grad_y[t] (0
 * for picks of nobody). Each may be NULL; rows is read for grad_weights only. The residual's is grad_y.
 */
int smx_combine_rows_grad(const void* grad_y, int64_t grad_y_stride, const void* rows,
                          int64_t rows_stride, int dtype, int64_t T, int64_t H, const int32_t* places,
                          int64_t k, const float* weights, void* grad_rows, float* grad_weights,
                          void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SPECMOE_MI355X_BLOCKS_H */
