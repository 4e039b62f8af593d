"""GELU and its slope where the normal distribution runs out (hip_layers.h):
the value at -5 is 1.4e-6 and has to keep its digits.  Arguments are exact:
planes of zeros leave z = beta, codes of zeros z = bias.

Tolerances (u = 2^-24).  Both hold e^(-z^2/2): its argument is off by u, and by
as much again and a quarter more where the exponential is one instruction of
the argument times log2 e, so the exponential by 1.2 z^2 u and a few u.  The
rest of the distribution Phi is sums of products and one quotient, taken as
good to 32 u: GELU z Phi within (2 z^2 + 36) u of its value; the slope Phi +
z phi within that of Phi, (2 z^2 + 16) u of z phi, and u of their sum.  An
exponential below the normal numbers may be 0, which moves a value by up to
2^-126 |z|.  An output type's rounding is on top.
"""
from __future__ import annotations

import math

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -122, torch.bfloat16: 2.0 ** -122, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
GELU = layers.ACTS["gelu"]


def arguments(count):
    z = torch.linspace(-13.0, 13.0, count, dtype=torch.float64)
    z[:12] = torch.tensor([-200.0, -90.0, -40.0, -14.0, -8.0, -6.0, -5.5, -5.0, -4.0, 5.0, 90.0,
                           200.0])
    return z.float().cuda()


def phi_of(z):
    """The normal distribution and its density in 64 bits."""
    return (0.5 * torch.special.erfc(-z / math.sqrt(2)),
            torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))


def check_values(y, z):
    zd = z.double()
    want = zd * phi_of(zd)[0]
    bound = ((2 * zd * zd + 36) * U + HALF_ULP[y.dtype]) * want.abs() + LEAST[y.dtype]
    over = (y.double() - want).abs() - bound
    worst = int(over.max(dim=-1).values.argmax()) if over.dim() > 1 else 0
    assert (over <= 0).all(), (worst, over.max().item())


def norm_space(images, pixels, channels, groups, dtype, backward):
    need = layers.group_norm_workspace_bytes(images, pixels, channels, groups,
                                             layers.DTYPES[dtype], backward)
    return torch.empty(need, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pixels", [1, 7, 20000])
def test_values_behind_a_norm(torch_cuda, dtype, pixels):
    """A plane that a workgroup holds, and one that takes chunks."""
    channels, groups = 512, 8
    z = arguments(channels)
    x = torch.zeros(1, pixels, channels, dtype=dtype, device="cuda")
    y = torch.empty_like(x)
    row = channels * x.element_size()
    assert layers.group_norm_device(x, pixels * row, row, None, z, y, None, None,
                                    norm_space(1, pixels, channels, groups, dtype, False), 1,
                                    pixels, channels, groups, 1e-5, GELU, layers.DTYPES[dtype],
                                    torch.cuda.current_stream()) == 1
    assert (y == y[:, :1]).all()
    check_values(y[0, 0], z)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 600, 40), (20, 600, 256), (300, 2048, 256)])
def test_values_behind_a_product(torch_cuda, dtype, m, n, k):
    """Few rows, and tiles staged through LDS."""
    z = arguments(n)
    kp = layers.mx4_padded(k)
    a_codes = torch.zeros(m, kp // 2, dtype=torch.uint8, device="cuda")
    w_codes = torch.full((n, kp // 2), 0x35, dtype=torch.uint8, device="cuda")
    a_scales, w_scales = (torch.full((r, kp // 32), 127, dtype=torch.uint8, device="cuda")
                          for r in (m, n))
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    assert layers.mx4_product_device(a_codes, a_scales, m, None, w_codes, w_scales, None, z, None,
                                     out, m, n, k, 1, GELU, layers.DTYPES[dtype],
                                     torch.cuda.current_stream()) == 1
    assert (out == out[:1]).all()
    check_values(out[0], z)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pixels", [1, 20000])
def test_slopes(torch_cuda, dtype, pixels):
    """dbeta of a gradient of ones at the first pixel alone: the slope itself."""
    channels, groups = 512, 8
    z = arguments(channels)
    x = torch.zeros(1, pixels, channels, dtype=dtype, device="cuda")
    dy = torch.zeros_like(x)
    dy[:, 0] = 1
    dx = torch.empty_like(x)
    mean, rstd = torch.zeros(1, groups, device="cuda"), torch.ones(1, groups, device="cuda")
    dgamma, dbeta = torch.empty(channels, device="cuda"), torch.empty(channels, device="cuda")
    row = channels * x.element_size()
    assert layers.group_norm_backward_device(
        x, pixels * row, row, dy, pixels * row, row, None, z, mean, rstd, dx, dgamma, dbeta,
        norm_space(1, pixels, channels, groups, dtype, True), 1, pixels, channels, groups, GELU,
        layers.DTYPES[dtype], torch.cuda.current_stream()) == 1
    zd = z.double()
    below, density = phi_of(zd)
    want = below + zd * density
    bound = ((2 * zd * zd + 36) * below + (2 * zd * zd + 16) * (zd * density).abs() +
             want.abs()) * U + 2.0 ** -122
    over = (dbeta.double() - want).abs() - bound
    assert (over <= 0).all(), (zd[over.argmax()].item(), over.max().item())
    assert (dgamma == 0).all()
