/*
 * specmoe_mi355x_products.h -- matrix products with an epilogue, dense and grouped by expert, and
 * their gradients: the products around and inside MoE blocks of other forms than the fused SwiGLU
 * page of specmoe_mi355x.h (experts with biases, GELU or ReLU experts, dense MLPs, projections), and
 * the training of any of them. Same library, same conventions: plain device pointers and sizes,
 * stream-ordered on `stream`, no host synchronisation, no device allocation (scratch is the
 * caller's workspace, 16-byte aligned), status codes of specmoe_mi355x.h. Calls are re-entrant for distinct
 * workspaces; a captured graph keeps using the workspace of its calls, so it needs one that no
 * other work uses while it runs. No counterpart in the reference, which leaves these products to
 * its framework.
 *
 *     z = x W^T + b           x [rows, K], W [Nw, K], b [Nw]
 *     y = residual + act(z)   y [rows, N]: Nw = N, or 2 N for SMX_ACT_SWIGLU, whose activation
 *                             silu(z[:, :N]) * z[:, N:] takes gate rows, then up rows of W
 *
 * Grouped: rows group_offsets[g] .. group_offsets[g + 1] - 1 use weight g and bias g, or with
 * weight_slots (int64 [G]) weight weight_slots[g] and bias weight_slots[g] of num_weights ones: the
 * slot map of an expert pool, whose pages [gate | up | down] hold the weight of gate and up at
 * their start (group_stride: page elements). group_offsets (int64 [G + 1], on the device) does
 * not decrease. Rows before the first bound, from the last one on, and of a group whose slot is
 * outside the pool are of no group: with fill_rest their y is the residual's row, or zero; without
 * it they are left as they were. Bounds outside [0, rows] are clamped to it.
 *
 * Element type of every tensor but z and the maps: `dtype`. Rows of x, residual, y and dy lie
 * *_stride elements apart (>= their length), elements of a row side by side. Products are summed
 * in fp32 and y is rounded once. Any rows >= 0, K, N >= 1 up to 2^30, pitches below 8 MiB, as many
 * output tiles as a grid holds (2^31 workgroups), a swiglu weight (of a group) below 2 GiB; any
 * alignment of elements (16-byte aligned rows are faster). Other sizes: SMX_ERR_UNSUPPORTED.
 */
#ifndef SPECMOE_MI355X_PRODUCTS_H
#define SPECMOE_MI355X_PRODUCTS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum smx_activation {
  SMX_ACT_NONE = 0,
  SMX_ACT_RELU = 1,
  SMX_ACT_GELU = 2,       /* z * (1 + erf(z / sqrt 2)) / 2 */
  SMX_ACT_GELU_TANH = 3,  /* z * (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2 */
  SMX_ACT_SILU = 4,       /* z / (1 + exp(-z)) */
  SMX_ACT_SWIGLU = 5
};

/* Bytes of workspace that smx_linear (G = 0) or smx_grouped_linear needs; 0 also for bad sizes. */
size_t smx_linear_workspace_size(int64_t rows, int64_t K, int64_t N, int64_t G, int activation,
                                 int dtype);

/*
 * y = residual + act(x W^T + b). weight [Nw, K], rows weight_stride elements apart. bias, residual:
 * may be NULL. preact: NULL, or fp32 [rows, Nw] (dense) that receives z for smx_linear_grad.
 * y may be the residual; it may not overlap anything else.
 */
int smx_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t K,
               const void* weight, int64_t weight_stride, int64_t N, const void* bias,
               int activation, const void* residual, int64_t residual_stride, void* y,
               int64_t y_stride, float* preact, void* workspace, size_t workspace_bytes,
               void* stream);

/* The same grouped. bias [num_weights, Nw]; num_weights = G without weight_slots. */
int smx_grouped_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t K,
                       const void* weight, int64_t weight_stride, int64_t group_stride,
                       int64_t num_weights, int64_t N, const void* bias, int activation,
                       const void* residual, int64_t residual_stride, const int64_t* group_offsets,
                       int64_t G, const int64_t* weight_slots, int fill_rest, void* y,
                       int64_t y_stride, float* preact, void* workspace, size_t workspace_bytes,
                       void* stream);

/* Bytes of workspace of the gradient calls (G = 0: dense); 0 for bad sizes. */
size_t smx_linear_grad_workspace_size(int64_t rows, int64_t K, int64_t N, int64_t G, int activation,
                                      int dtype);

/*
 * Gradients of smx_linear for the gradient dy of y: with dz = dy * act'(z),
 *     grad_x = dz W, grad_weight = dz^T x, grad_bias = the column sums of dz
 * (the residual's is dy), each dense, in `dtype`, or NULL where it is not wanted. preact: the
 * forward call's z (not read for SMX_ACT_NONE). dz is summed into grad_bias in fp32 and rounded to
 * `dtype` as an operand of the two products. Sums run in a fixed order.
 */
int smx_linear_grad(const void* dy, int64_t dy_stride, const float* preact, const void* x,
                    int64_t x_stride, int dtype, int64_t rows, int64_t K, const void* weight,
                    int64_t weight_stride, int64_t N, int activation, void* grad_x,
                    void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                    void* stream);

/*
 * The same grouped: grad_x is zero in rows of no group, grad_weight [G, Nw, K] and grad_bias
 * [G, Nw] in groups without rows. With weight_slots only grad_x is available (two groups may share a slot).
 */
int smx_grouped_linear_grad(const void* dy, int64_t dy_stride, const float* preact, const void* x,
                            int64_t x_stride, int dtype, int64_t rows, int64_t K,
                            const void* weight, int64_t weight_stride, int64_t group_stride,
                            int64_t num_weights, int64_t N, int activation,
                            const int64_t* group_offsets, int64_t G, const int64_t* weight_slots,
                            void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                            size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SPECMOE_MI355X_PRODUCTS_H */
