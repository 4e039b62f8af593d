/*
 * Layers behind the 618M actor's sensor preparation
 * (tb_hip_actor_inputs_device in hip_features.h), offered by the gfx950
 * backend (libturbinator_hip):
 *   - group norm with an activation over channels-last planes, forward and
 *     backward (the convolution stems);
 *   - routing of tokens to experts, forward and backward, and the order of
 *     the choices by expert;
 *   - microscaled 4-bit floating point: quantisation, its values, and
 *     products on the scaled matrix instructions, dense or per expert.
 * All pointers are device pointers.  All entries are asynchronous on `stream`
 * (a hipStream_t as void*, NULL = null stream), allocate nothing and return 1
 * iff the launches were accepted, 0 on invalid arguments (nothing is launched
 * then).  Strides are bytes.  Outputs must not overlap inputs, each other or
 * the workspace.  Results do not depend on the run: no sum's order does.
 */
#ifndef TURBINATOR_HIP_LAYERS_H
#define TURBINATOR_HIP_LAYERS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the `dtype` arguments, activations of the `act` arguments
 * (SiLU z / (1 + e^-z); GELU z Phi(z), Phi the normal distribution) and
 * scores of the `score` arguments. */
enum { TB_HIP_F32 = 0, TB_HIP_BF16 = 1, TB_HIP_F16 = 2 };
enum { TB_HIP_ACT_NONE = 0, TB_HIP_ACT_SILU = 1, TB_HIP_ACT_GELU = 2 };
enum { TB_HIP_SCORE_SOFTMAX = 0, TB_HIP_SCORE_SIGMOID = 1 };

enum {
    TB_HIP_NORM_MAX_GROUP = 1024,  /* channels of one group */
    TB_HIP_NORM_MAX_CHANNELS = 65536,
    TB_HIP_ROUTE_MAX_EXPERTS = 1024,
    TB_HIP_ROUTE_MAX_K = 32,
    TB_HIP_MX4_BLOCK = 32          /* values that share a scale */
};

/* y = act((x - mean) rstd gamma + beta) over channels-last planes: `images`
 * images of `pixels` pixels of `channels` channels, mean and variance (biased)
 * over the pixels and the channels / groups consecutive channels of a group.
 * x: element (i, p, c) lies at byte i image_stride + p pixel_stride + c size;
 * y is dense.  Sums and statistics are held in 32 bits, the variance as the
 * mean square of the deviations; y is rounded once.  gamma and beta (fp32,
 * [channels]) may be NULL (1 and 0).  mean and rstd ([images, groups] fp32)
 * may be NULL; the backward pass reads them.
 * workspace: tb_hip_group_norm_workspace_bytes(..., backward 0) bytes, 16-byte
 * aligned.
 * Returns 0 for NULL x or y, a workspace that is NULL or misaligned,
 * images, pixels, channels or groups 0 or images or pixels above 0x7fffffff,
 * channels above TB_HIP_NORM_MAX_CHANNELS or not a multiple of groups, a group
 * above TB_HIP_NORM_MAX_GROUP channels, x, y or strides that are not multiples
 * of the element's size, an unknown act or dtype, or an eps that is not
 * positive and finite. */
int tb_hip_group_norm_device(const void *x, size_t image_stride, size_t pixel_stride,
                             const float *gamma, const float *beta, void *y, float *mean,
                             float *rstd, void *workspace, size_t images, size_t pixels,
                             int channels, int groups, float eps, int act, int dtype,
                             void *stream);

/* The gradients of tb_hip_group_norm_device for the gradient dy of y: dx
 * (dense, the type of x), dgamma and dbeta (fp32 [channels], both or neither
 * NULL).  x and dy are strided like x above (a stride may be 0: a gradient
 * that is the same for every pixel); gamma and beta as in the forward pass;
 * mean and rstd are its outputs.  With u = dy act'(z) gamma and h = (x - mean)
 * rstd: dx = rstd (u - mean(u) - h mean(u h)), the means over a group.
 * workspace: tb_hip_group_norm_workspace_bytes(..., backward 1) bytes.
 * Returns 0 as above, and for NULL dy, mean, rstd, dx or workspace. */
int tb_hip_group_norm_backward_device(const void *x, size_t x_image_stride,
                                      size_t x_pixel_stride, const void *dy,
                                      size_t dy_image_stride, size_t dy_pixel_stride,
                                      const float *gamma, const float *beta, const float *mean,
                                      const float *rstd, void *dx, float *dgamma, float *dbeta,
                                      void *workspace, size_t images, size_t pixels,
                                      int channels, int groups, int act, int dtype,
                                      void *stream);

/* Workspace of the entries above for these sizes, enough for any strides and
 * alignment; 0 for sizes they refuse. */
size_t tb_hip_group_norm_workspace_bytes(size_t images, size_t pixels, int channels, int groups,
                                         int dtype, int backward);

/* Routing: for each token (row of `logits`, row_stride bytes apart, n_experts
 * values) the k experts of the highest keys, best first, equal keys in the
 * order of their index, and their weights.
 *   scores   s = softmax(logits) or sigmoid(logits), in 32 bits
 *   keys     the logits, or s + bias with a bias ([n_experts] fp32, for
 *            balance: it chooses and does not weigh)
 *   groups   n_experts / groups consecutive experts each; only the
 *            groups_kept best groups' experts are chosen from, a group's
 *            standing being its best key, with a bias the sum of its two best
 *   weights  scale s, with renormalise scale s / (sum of the token's chosen s)
 *            (0 where that sum is 0)
 * An expert whose logit or key is -inf is never chosen; where too few are
 * left the remaining experts are -1 and their weights 0, and so is the whole
 * row of a token whose `valid` byte (nullable, [tokens]) is 0, whose logits
 * are not read.  NaN keys count as the highest.  An expert with a NaN logit has
 * a NaN weight, with softmax or renormalise the whole row; a NaN in the bias
 * chooses, and does not weigh either.
 * experts [tokens, k] int32, weights [tokens, k] fp32.
 * Returns 0 for NULL logits, experts or weights, tokens 0 or tokens * k above
 * 0x7fffffff, n_experts outside 1..TB_HIP_ROUTE_MAX_EXPERTS, k outside
 * 1..min(n_experts, TB_HIP_ROUTE_MAX_K), groups that do not divide n_experts,
 * groups_kept outside 1..groups or of fewer than k experts together, an
 * unknown score or dtype, logits or a stride off the element's size. */
int tb_hip_route_device(const void *logits, size_t row_stride, const float *bias,
                        const unsigned char *valid, int *experts, float *weights, size_t tokens,
                        int n_experts, int k, int groups, int groups_kept, int score,
                        int renormalise, float scale, int dtype, void *stream);

/* The gradient dlogits (dense, the type of logits) of the weights for their
 * gradient dweights [tokens, k], the choice held fixed.  experts as the
 * forward pass chose them; those outside 0..n_experts-1 (-1) have no part,
 * and a row of them alone has a zero gradient and is not read.  Same argument
 * rules. */
int tb_hip_route_backward_device(const void *logits, size_t row_stride, const int *experts,
                                 const float *dweights, void *dlogits, size_t tokens,
                                 int n_experts, int k, int score, int renormalise, float scale,
                                 int dtype, void *stream);

/* The tokens * k choices in the order of their experts, equal experts in the
 * order of the choices (choice c = token c / k):
 *   offsets [n_experts + 1]  expert x has rows offsets[x] .. offsets[x+1]-1
 *   tokens_out [tokens * k]  the token of each row, -1 behind the last expert's
 *   positions [tokens, k]    the row of each choice, -1 for a choice outside
 *                            0..n_experts-1
 *   row_weights [tokens * k] the weight of each row, 0 behind the last
 *                            expert's; weights and row_weights may be NULL
 *                            together
 * workspace: tb_hip_expert_order_workspace_bytes(...) bytes, 16-byte aligned.
 * Returns 0 for NULL pointers otherwise, tokens 0 or tokens * k above
 * 0x7fffffff, n_experts outside 1..TB_HIP_ROUTE_MAX_EXPERTS or k outside
 * 1..TB_HIP_ROUTE_MAX_K. */
int tb_hip_expert_order_device(const int *experts, const float *weights, int *offsets,
                               int *tokens_out, int *positions, float *row_weights,
                               void *workspace, size_t tokens, int n_experts, int k,
                               void *stream);
size_t tb_hip_expert_order_workspace_bytes(size_t tokens, int n_experts, int k);

/* Microscaled 4-bit floating point (the OCP MX format MXFP4): 32 consecutive
 * values of a row share a scale 2^(s - 127), s one byte, and are held as sign,
 * two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6).  A row
 * of k values is padded with zeros to kp = tb_hip_mx4_padded(k), whole 128s:
 * codes [rows, kp / 2] bytes, the even value in the low half; scales
 * [rows, kp / 32] bytes.  codes must be 16-byte, scales 4-byte aligned.
 *
 * Quantisation: s - 127 = floor(log2(largest magnitude)) - 2, at least -127;
 * values rounded to nearest, ties to even, magnitudes above 6 to 6.  A block
 * that holds an Inf or a NaN has s = 255 (NaN) and zero codes. */
size_t tb_hip_mx4_padded(size_t k);
int tb_hip_mx4_quantise_device(const void *x, size_t row_stride, void *codes, void *scales,
                               size_t rows, size_t k, int dtype, void *stream);

/* The values [rows, k] (dense) that codes and scales stand for, rounded to
 * the type: f16 can round or overflow, f32 and bf16 can overflow for scales of
 * 253 and 254, which quantisation does not give.
 * Both return 0 for NULL pointers, rows or k 0 or above 0x7fffffff, an
 * unknown dtype or misaligned pointers or stride. */
int tb_hip_mx4_values_device(const void *codes, const void *scales, void *values, size_t rows,
                             size_t k, int dtype, void *stream);

/* out[r] = act(A[a(r)] W[x(r)]^T + bias[x(r)]) row_scale[r]: products of
 * quantised rows, summed in 32 bits and rounded once.  A: a_rows rows of k.
 * W: experts * n rows of k, bias [experts, n] fp32 (nullable), row_scale [m]
 * fp32 (nullable).
 *   a(r) = rows[r], or r with rows NULL (then m = a_rows)
 *   x(r) = the expert with offsets[x] <= r < offsets[x+1]; experts = 1 and
 *          offsets NULL for one dense product
 * Rows that belong to no expert, or whose rows[r] is outside 0..a_rows-1,
 * come out as 0.  offsets must not decrease; entries are taken as at least 0
 * and at most m.  out [m, n] is dense.
 * Returns 0 for other NULL pointers, m, n, k or a_rows 0 or above 0x7fffffff,
 * experts outside 1..TB_HIP_ROUTE_MAX_EXPERTS or above 1 without offsets,
 * experts * n above 0x7fffffff, m * n above 2^38, rows NULL with m other than
 * a_rows, an unknown act or dtype, or misaligned pointers. */
int tb_hip_mx4_product_device(const void *a_codes, const void *a_scales, size_t a_rows,
                              const int *rows, const void *w_codes, const void *w_scales,
                              const int *offsets, const float *bias, const float *row_scale,
                              void *out, size_t m, size_t n, size_t k, int experts, int act,
                              int dtype, void *stream);

#ifdef __cplusplus
}
#endif

#endif
