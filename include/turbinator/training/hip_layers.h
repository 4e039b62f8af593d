/*
 * Layers behind the 618M actor's sensor preparation
 * (tb_hip_actor_inputs_device in hip_features.h), offered by the gfx950
 * backend (libturbinator_hip):
 *   - group norm with an activation over channels-last planes, forward and
 *     backward (the convolution stems);
 *   - routing of tokens to experts, forward and backward, and the order of
 *     the choices by expert.
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
    TB_HIP_ROUTE_MAX_K = 32
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
 * above TB_HIP_NORM_MAX_GROUP channels, x, y or strides that are not multiples of the element's size, an
 * unknown act or dtype, or an eps that is not positive and finite. */
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
 * are not read.  NaN keys count as the highest and give NaN weights.
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

#ifdef __cplusplus
}
#endif

#endif
