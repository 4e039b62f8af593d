"""Python mirror of the layer entries (include/turbinator/training/hip_layers.h).

Functions return 1 on success and 0 on refused arguments, exactly like the C
entries they call; none allocates or waits.  Device arguments accept torch
tensors on the GPU or raw device addresses; strides are bytes; `dtype`, `act`
and `score` take the values of DTYPES, ACTS and SCORES.
"""
from __future__ import annotations

from .features import _dev, _stream
from .native import hip_lib

try:
    import torch
    DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
except ImportError:  # raw addresses need no torch
    DTYPES = {}
DTYPES.update({"f32": 0, "bf16": 1, "f16": 2})
ACTS = {"none": 0, "silu": 1, "gelu": 2}
SCORES = {"softmax": 0, "sigmoid": 1}
MX4_BLOCK = 32


def group_norm_workspace_bytes(images: int, pixels: int, channels: int, groups: int, dtype: int,
                               backward: bool = False) -> int:
    return hip_lib().tb_hip_group_norm_workspace_bytes(images, pixels, channels, groups, dtype,
                                                       1 if backward else 0)


def group_norm_device(x, image_stride: int, pixel_stride: int, gamma, beta, y, mean, rstd,
                      workspace, images: int, pixels: int, channels: int, groups: int,
                      eps: float, act: int, dtype: int, stream=None) -> int:
    """tb_hip_group_norm_device."""
    return hip_lib().tb_hip_group_norm_device(
        _dev(x), image_stride, pixel_stride, _dev(gamma), _dev(beta), _dev(y), _dev(mean),
        _dev(rstd), _dev(workspace), images, pixels, channels, groups, eps, act, dtype,
        _stream(stream))


def group_norm_backward_device(x, x_image_stride: int, x_pixel_stride: int, dy,
                               dy_image_stride: int, dy_pixel_stride: int, gamma, beta, mean,
                               rstd, dx, dgamma, dbeta, workspace, images: int, pixels: int,
                               channels: int, groups: int, act: int, dtype: int,
                               stream=None) -> int:
    """tb_hip_group_norm_backward_device."""
    return hip_lib().tb_hip_group_norm_backward_device(
        _dev(x), x_image_stride, x_pixel_stride, _dev(dy), dy_image_stride, dy_pixel_stride,
        _dev(gamma), _dev(beta), _dev(mean), _dev(rstd), _dev(dx), _dev(dgamma), _dev(dbeta),
        _dev(workspace), images, pixels, channels, groups, act, dtype, _stream(stream))


def route_device(logits, row_stride: int, bias, valid, experts, weights, tokens: int,
                 n_experts: int, k: int, groups: int, groups_kept: int, score: int,
                 renormalise: bool, scale: float, dtype: int, stream=None) -> int:
    """tb_hip_route_device."""
    return hip_lib().tb_hip_route_device(
        _dev(logits), row_stride, _dev(bias), _dev(valid), _dev(experts), _dev(weights), tokens,
        n_experts, k, groups, groups_kept, score, 1 if renormalise else 0, scale, dtype,
        _stream(stream))


def route_backward_device(logits, row_stride: int, experts, dweights, dlogits, tokens: int,
                          n_experts: int, k: int, score: int, renormalise: bool, scale: float,
                          dtype: int, stream=None) -> int:
    """tb_hip_route_backward_device."""
    return hip_lib().tb_hip_route_backward_device(
        _dev(logits), row_stride, _dev(experts), _dev(dweights), _dev(dlogits), tokens,
        n_experts, k, score, 1 if renormalise else 0, scale, dtype, _stream(stream))


def expert_order_workspace_bytes(tokens: int, n_experts: int, k: int) -> int:
    return hip_lib().tb_hip_expert_order_workspace_bytes(tokens, n_experts, k)


def expert_order_device(experts, weights, offsets, tokens_out, positions, row_weights, workspace,
                        tokens: int, n_experts: int, k: int, stream=None) -> int:
    """tb_hip_expert_order_device."""
    return hip_lib().tb_hip_expert_order_device(
        _dev(experts), _dev(weights), _dev(offsets), _dev(tokens_out), _dev(positions),
        _dev(row_weights), _dev(workspace), tokens, n_experts, k, _stream(stream))


def mx4_padded(k: int) -> int:
    return hip_lib().tb_hip_mx4_padded(k)


def mx4_quantise_device(x, row_stride: int, codes, scales, rows: int, k: int, dtype: int,
                        stream=None) -> int:
    """tb_hip_mx4_quantise_device."""
    return hip_lib().tb_hip_mx4_quantise_device(_dev(x), row_stride, _dev(codes), _dev(scales),
                                                rows, k, dtype, _stream(stream))


def mx4_values_device(codes, scales, values, rows: int, k: int, dtype: int, stream=None) -> int:
    """tb_hip_mx4_values_device."""
    return hip_lib().tb_hip_mx4_values_device(_dev(codes), _dev(scales), _dev(values), rows, k,
                                              dtype, _stream(stream))


def mx4_product_device(a_codes, a_scales, a_rows: int, rows, w_codes, w_scales, offsets, bias,
                       row_scale, out, m: int, n: int, k: int, experts: int, act: int,
                       dtype: int, stream=None) -> int:
    """tb_hip_mx4_product_device."""
    return hip_lib().tb_hip_mx4_product_device(
        _dev(a_codes), _dev(a_scales), a_rows, _dev(rows), _dev(w_codes), _dev(w_scales),
        _dev(offsets), _dev(bias), _dev(row_scale), _dev(out), m, n, k, experts, act, dtype,
        _stream(stream))


__all__ = ["DTYPES", "ACTS", "SCORES", "MX4_BLOCK", "group_norm_workspace_bytes",
           "group_norm_device", "group_norm_backward_device", "route_device",
           "route_backward_device", "expert_order_workspace_bytes", "expert_order_device",
           "mx4_padded", "mx4_quantise_device", "mx4_values_device", "mx4_product_device"]
