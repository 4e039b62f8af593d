"""Group norm with an activation (hip_layers.h) against the formula in 64 bits:
every type and activation, one pixel and many, odd channels and groups, slices
of wider rows, planes longer than one chunk, NaN in one image, large means,
gradients against the formula's and against differences.

Tolerances.  u is half an ulp of 32 bits (2^-24).  Sums run over at most a few
dozen sequential terms and a tree, so the mean is within 64 u of the mean
magnitude and the variance within 64 u relative; z inherits 64 u of
(|x| + |mean|) rstd |gamma| and 64 u of its own size, and the activations'
slopes stay below 1.13.  The output type's rounding (half an ulp) is on top.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def act(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return torch.nn.functional.gelu(z)
    return z


def oracle(x, gamma, beta, groups, name):
    """y, mean, rstd in 64 bits; x [n, p, c]."""
    n, p, c = x.shape
    v = x.reshape(n, p, groups, c // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True).add(EPS).rsqrt()
    z = ((v - mean) * rstd).reshape(n, p, c)
    z = z * (1 if gamma is None else gamma) + (0 if beta is None else beta)
    return act(z, name), z, mean.reshape(n, groups), rstd.reshape(n, groups)


def planes(seed, n, p, c, dtype, pitch=None, gap=0, mean=0.5):
    """A [n, p, c] slice of [n, p + gap, pitch] rows, NaN outside it."""
    g = torch.Generator().manual_seed(seed)
    pitch = pitch or c
    wide = torch.full((n, p + gap, pitch), float("nan"))
    off = pitch - c
    wide[:, :p, off:] = torch.randn((n, p, c), generator=g) * (0.5 + torch.rand(c, generator=g))
    wide[:, :p, off:] += mean * torch.randn(c, generator=g)
    return wide.to(dtype).cuda()[:, :p, off:]


def params(seed, c):
    g = torch.Generator().manual_seed(seed + 1000)
    return (1 + 0.3 * torch.randn(c, generator=g)).cuda(), (0.3 * torch.randn(c, generator=g)).cuda()


def strides(x):
    return x.stride(0) * x.element_size(), x.stride(1) * x.element_size()


def workspace(n, p, c, groups, dtype, backward):
    need = layers.group_norm_workspace_bytes(n, p, c, groups, layers.DTYPES[dtype], backward)
    # The bytes behind it hold a pattern that no call may touch.
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    return ws, need


def forward(x, gamma, beta, groups, name, eps=EPS, stream=None):
    n, p, c = x.shape
    y = torch.full((n, p, c), 7.0, dtype=x.dtype, device="cuda")
    mean, rstd = (torch.full((n, groups), 7.0, device="cuda") for _ in range(2))
    ws, need = workspace(n, p, c, groups, x.dtype, False)
    assert layers.group_norm_device(x, *strides(x), gamma, beta, y, mean, rstd, ws, n, p, c,
                                    groups, eps, layers.ACTS[name], layers.DTYPES[x.dtype],
                                    stream or torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (ws[need:] == 0x5a).all()
    return y, mean, rstd


def forward_bound(x, gamma, z, mean, rstd, groups, dtype, y):
    n, p, c = x.shape
    size = (x.abs().reshape(n, p, groups, -1) + mean.abs()[:, None, :, None]) * \
        rstd[:, None, :, None]
    size = size.reshape(n, p, c) * (1 if gamma is None else gamma.abs()) + z.abs() + 1
    return 1.13 * 64 * U * size + HALF_ULP[dtype] * y.abs() + LEAST[dtype]


def check_forward(x, gamma, beta, groups, name):
    y, mean, rstd = forward(x, gamma, beta, groups, name)
    xd = x.double()
    gd, bd = (None if t is None else t.double() for t in (gamma, beta))
    want, z, wmean, wrstd = oracle(xd, gd, bd, groups, name)
    size = xd.abs().reshape(x.shape[0], x.shape[1], groups, -1).mean(dim=(1, 3))
    assert ((mean.double() - wmean).abs() <= 64 * U * size + 1e-38).all()
    # A mean that is off shifts every deviation: u (size rstd)^2 of the variance.
    assert ((rstd.double() - wrstd).abs() <= 64 * U * wrstd * (1 + (size * wrstd) ** 2)).all()
    bound = forward_bound(xd, gd, z, wmean, wrstd, groups, x.dtype, want)
    over = ((y.double() - want).abs() - bound).max().item()
    assert over <= 0, over


SHAPES = [
    # images, pixels, channels, groups
    (1, 1, 1, 1), (3, 1, 64, 8), (2, 17, 6, 3), (5, 33, 7, 7), (1, 2048, 64, 8),
    (4, 300, 48, 6), (2, 1000, 24, 1), (3, 65, 320, 32), (2, 40, 1023, 1), (2, 9, 2048, 2),
    (1, 5000, 12, 2), (7, 129, 160, 4), (2, 31, 130, 13), (1, 40000, 8, 2), (2, 20000, 64, 4),
    (300, 16, 32, 8), (1, 7, 4092, 4),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(torch_cuda, shape, dtype):
    n, p, c, groups = shape
    gamma, beta = params(c, c)
    name = ["none", "silu", "gelu"][(n + p + c) % 3]
    print(shape, dtype, name, flush=True)
    check_forward(planes(p + c, n, p, c, dtype), gamma, beta, groups, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
@pytest.mark.parametrize("pitch,gap", [(32, 0), (36, 3), (33, 1), (48, 0), (64, 5)])
def test_forward_strided(torch_cuda, dtype, name, pitch, gap):
    x = planes(pitch, 3, 70, 32, dtype, pitch, gap)
    gamma, beta = params(5, 32)
    check_forward(x, gamma, beta, 4, name)
    check_forward(x, None, None, 8, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_large_means(torch_cuda, dtype):
    """Means a hundred times the deviation: no cancelling mean of squares."""
    check_forward(planes(3, 2, 600, 32, dtype, mean=100.0), None, None, 8, "none")


@pytest.mark.parametrize("pixels", [5, 1500, 30000])
def test_constant_planes(torch_cuda, pixels):
    """No deviation at all: y is act(beta) and rstd 1 / sqrt(eps)."""
    x = torch.full((2, pixels, 16), 3.0, device="cuda")
    gamma, beta = params(1, 16)
    y, mean, rstd = forward(x, gamma, beta, 4, "silu")
    assert (mean == 3.0).all()
    assert ((rstd.double() * EPS ** 0.5 - 1).abs() < 4 * U).all()
    want = act(beta.double(), "silu")
    assert ((y.double() - want).abs() <= 8 * U * (1 + want.abs())).all()


def test_nan_and_inf_stay_in_their_group(torch_cuda):
    x = planes(9, 3, 50, 32, torch.float32)
    x[1, 7, 3] = float("nan")
    x[2, 9, 30] = float("inf")
    y, mean, rstd = forward(x, None, None, 4, "silu")
    bad = torch.zeros((3, 4), dtype=torch.bool, device="cuda")
    bad[1, 0] = bad[2, 3] = True
    assert (torch.isnan(rstd) == bad).all()
    per = torch.isnan(y).reshape(3, 50, 4, 8).all(dim=3).all(dim=1)
    some = torch.isnan(y).reshape(3, 50, 4, 8).any(dim=3).any(dim=1)
    assert (per == bad).all() and (some == bad).all()


def test_extreme_arguments_of_the_activations(torch_cuda):
    """Beta far out: SiLU and GELU run to z and to 0 without NaN."""
    x = planes(4, 1, 64, 8, torch.float32)
    beta = torch.tensor([-200.0, -90.0, -20.0, -5.0, 5.0, 20.0, 90.0, 200.0], device="cuda")
    for name in ("silu", "gelu"):
        y, _, _ = forward(x, None, beta, 8, name)
        want = oracle(x.double(), None, beta.double(), 8, name)[0]
        assert torch.isfinite(y).all()
        assert ((y.double() - want).abs() <= 1e-4 * want.abs() + 64 * U * 200).all()


def test_other_stream(torch_cuda):
    x = planes(2, 4, 500, 64, torch.bfloat16)
    gamma, beta = params(2, 64)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    first = forward(x, gamma, beta, 8, "silu")
    second = forward(x, gamma, beta, 8, "silu", stream=side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_optional_outputs(torch_cuda):
    x = planes(2, 4, 500, 64, torch.float32)
    y = torch.empty_like(x)
    ws, _ = workspace(4, 500, 64, 8, x.dtype, False)
    assert layers.group_norm_device(x, *strides(x), None, None, y, None, None, ws, 4, 500, 64, 8,
                                    EPS, 1, 0, torch.cuda.current_stream()) == 1
    assert torch.equal(y, forward(x, None, None, 8, "silu")[0])


# --------------------------------------------------------------------------
# Backward


def gradients(x, dy, gamma, beta, mean, rstd, groups, name, params_too=True):
    n, p, c = x.shape
    dx = torch.full((n, p, c), 7.0, dtype=x.dtype, device="cuda")
    dgamma, dbeta = (torch.full((c,), 7.0, device="cuda") for _ in range(2))
    ws, need = workspace(n, p, c, groups, x.dtype, True)
    assert layers.group_norm_backward_device(
        x, *strides(x), dy, *strides(dy), gamma, beta, mean, rstd, dx,
        dgamma if params_too else None, dbeta if params_too else None, ws, n, p, c, groups,
        layers.ACTS[name], layers.DTYPES[x.dtype], torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (ws[need:] == 0x5a).all()
    return dx, dgamma, dbeta


def check_backward(x, dy, gamma, beta, groups, name):
    n, p, c = x.shape
    _, mean, rstd = forward(x, gamma, beta, groups, name)
    dx, dgamma, dbeta = gradients(x, dy, gamma, beta, mean, rstd, groups, name)
    # The formula at the statistics that the call was given.
    m, r = (t.double().repeat_interleave(c // groups, dim=1)[:, None] for t in (mean, rstd))
    g = torch.ones(c, dtype=torch.float64, device="cuda") if gamma is None else gamma.double()
    b = torch.zeros_like(g) if beta is None else beta.double()
    h = ((x.double() - m) * r)
    z = (h * g + b).requires_grad_()
    slope, = torch.autograd.grad(act(z, name).sum(), z)
    u = dy.double() * slope
    # u is off by 64 u of itself and by the slope's change over z's error.
    du = 64 * U * (u.abs() + dy.double().abs() * ((x.double().abs() + m.abs()) * r * g.abs() +
                                                  z.detach().abs() + 1))
    dh = 8 * U * (x.double().abs() + m.abs()) * r

    def mean_of(v):
        return v.reshape(n, p, groups, -1).mean(dim=(1, 3)).repeat_interleave(
            c // groups, dim=1)[:, None]

    ug = u * g
    m1, m2 = mean_of(ug), mean_of(ug * h)
    want = r * (ug - m1 - h * m2)
    dm1 = mean_of(du * g.abs()) + 64 * U * mean_of(ug.abs())
    dm2 = mean_of(du * g.abs() * h.abs() + ug.abs() * dh) + 64 * U * mean_of((ug * h).abs())
    bound = r * (du * g.abs() + dm1 + h.abs() * dm2 + dh * m2.abs() +
                 8 * U * (ug.abs() + m1.abs() + (h * m2).abs()))
    bound = bound + HALF_ULP[x.dtype] * want.abs() + LEAST[x.dtype]
    over = ((dx.double() - want).abs() - bound).max().item()
    assert over <= 0, over
    assert ((dbeta.double() - u.sum(dim=(0, 1))).abs() <=
            (du + 64 * U * u.abs()).sum(dim=(0, 1)) + 1e-38).all()
    assert ((dgamma.double() - (u * h).sum(dim=(0, 1))).abs() <=
            (du * h.abs() + u.abs() * dh + 64 * U * (u * h).abs()).sum(dim=(0, 1)) + 1e-38).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(torch_cuda, shape, dtype):
    n, p, c, groups = shape
    gamma, beta = params(c, c)
    name = ["none", "silu", "gelu"][(n + p + c + 1) % 3]
    print(shape, dtype, name, flush=True)
    check_backward(planes(p, n, p, c, dtype), planes(p + 1, n, p, c, dtype), gamma, beta, groups,
                   name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
@pytest.mark.parametrize("pitch,gap", [(36, 3), (33, 1), (64, 5)])
def test_backward_strided(torch_cuda, dtype, name, pitch, gap):
    x = planes(pitch, 3, 70, 32, dtype, pitch, gap)
    dy = planes(pitch + 1, 3, 70, 32, dtype, 40, 2)
    gamma, beta = params(5, 32)
    check_backward(x, dy, gamma, beta, 4, name)
    check_backward(x, dy, None, None, 8, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_backward_of_a_broadcast_gradient(torch_cuda, dtype):
    """dy the same for every pixel (stride 0), as the mean over pixels leaves it."""
    x = planes(8, 5, 90, 32, dtype)
    dy = planes(9, 5, 1, 32, dtype).expand(5, 90, 32)
    assert dy.stride(1) == 0
    gamma, beta = params(6, 32)
    check_backward(x, dy, gamma, beta, 8, "silu")
    one = planes(9, 1, 1, 32, dtype).expand(5, 90, 32)
    check_backward(x, one, gamma, beta, 8, "gelu")


def test_backward_without_parameters(torch_cuda):
    x, dy = planes(8, 5, 90, 32, torch.float32), planes(9, 5, 90, 32, torch.float32)
    _, mean, rstd = forward(x, None, None, 8, "silu")
    with_them = gradients(x, dy, None, None, mean, rstd, 8, "silu")
    without = gradients(x, dy, None, None, mean, rstd, 8, "silu", params_too=False)
    assert torch.equal(with_them[0], without[0])
    assert (without[1] == 7).all() and (without[2] == 7).all()


def test_backward_repeats_bit_for_bit(torch_cuda):
    x, dy = planes(8, 700, 64, 32, torch.bfloat16), planes(9, 700, 64, 32, torch.bfloat16)
    gamma, beta = params(6, 32)
    _, mean, rstd = forward(x, gamma, beta, 8, "silu")
    first = gradients(x, dy, gamma, beta, mean, rstd, 8, "silu")
    for _ in range(3):
        for a, b in zip(first, gradients(x, dy, gamma, beta, mean, rstd, 8, "silu")):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
def test_gradient_against_differences(torch_cuda, name):
    """Along random directions of x, gamma and beta, against central
    differences of the 64-bit forward pass: steps of 1e-5 are off by about
    1e-10 of the loss's size, the gradients by the 32-bit sums' 1e-5."""
    n, p, c, groups = 2, 40, 24, 4
    x, dy = planes(11, n, p, c, torch.float32), planes(12, n, p, c, torch.float32)
    gamma, beta = params(7, c)
    _, mean, rstd = forward(x, gamma, beta, groups, name)
    grads = gradients(x, dy, gamma, beta, mean, rstd, groups, name)
    at = [t.double() for t in (x, gamma, beta)]
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        way = [torch.randn(t.shape, generator=g, dtype=torch.float64).cuda() for t in at]

        def loss(h):
            xx, gg, bb = (t + h * w for t, w in zip(at, way))
            return (oracle(xx, gg, bb, groups, name)[0] * dy.double()).sum().item()

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        terms = [gr.double() * w for gr, w in zip(grads, way)]
        got = sum(t.sum().item() for t in terms)
        size = sum(t.abs().sum().item() for t in terms)
        assert abs(got - slope) <= 1e-5 * size, (got, slope, size)


def test_refusals(torch_cuda):
    x = torch.zeros((2, 4, 8), device="cuda")
    out = torch.full((2, 4, 8), 7.0, device="cuda")
    stat = torch.zeros((2, 2), device="cuda")
    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    good = dict(x=x, si=128, sp=32, y=out, ws=ws, n=2, p=4, c=8, g=2, eps=1e-5, act=1, dt=0)

    def call(**over):
        a = {**good, **over}
        return layers.group_norm_device(a["x"], a["si"], a["sp"], None, None, a["y"], None, None,
                                        a["ws"], a["n"], a["p"], a["c"], a["g"], a["eps"],
                                        a["act"], a["dt"], torch.cuda.current_stream())

    def back(**over):
        a = {**good, "dy": x, "mean": stat, "rstd": stat, "dg": None, "db": None, **over}
        return layers.group_norm_backward_device(
            a["x"], a["si"], a["sp"], a["dy"], 128, 32, None, None, a["mean"], a["rstd"], a["y"],
            a["dg"], a["db"], a["ws"], a["n"], a["p"], a["c"], a["g"], a["act"], a["dt"],
            torch.cuda.current_stream())

    bad = [dict(x=None), dict(y=None), dict(ws=None), dict(n=0), dict(p=0), dict(c=0), dict(g=0),
           dict(g=3), dict(c=-8), dict(g=-2), dict(n=0x80000000), dict(p=0x80000000),
           dict(act=3), dict(act=-1), dict(dt=3), dict(dt=-1), dict(si=130), dict(sp=30),
           dict(x=x.data_ptr() + 2), dict(y=out.data_ptr() + 2), dict(ws=ws.data_ptr() + 4),
           dict(c=2050, g=2, sp=8200), dict(c=131072, g=1024)]
    for over in bad:
        assert call(**over) == 0, over
        assert back(**over) == 0, over
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        assert call(eps=eps) == 0
    for over in (dict(dy=None), dict(mean=None), dict(rstd=None), dict(dg=stat),
                 dict(db=stat), dict(dy=x.data_ptr() + 2)):
        assert back(**over) == 0, over
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert call() == 1 and back() == 1
    torch.cuda.synchronize()


def test_plane_longer_than_its_chunks(torch_cuda):
    """Five million pixels: chunks of several sweeps, joined twice."""
    gamma, beta = params(3, 2)
    x, dy = (planes(s, 1, 5_000_000, 2, torch.float32) for s in (21, 22))
    check_forward(x, gamma, beta, 1, "silu")
    check_backward(x, dy, gamma, beta, 1, "silu")
