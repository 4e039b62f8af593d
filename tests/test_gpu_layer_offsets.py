"""The layer entries where byte offsets pass 32 bits: rows, pixels and images
far apart, and matrices and outputs above 4 GiB.  Each is the same call on near
data, bit for bit: the kernels take their variant by sizes and alignment, which
are the same, and the products are of small integers, whose sums are exact in
32 bits in any order."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers  # noqa: E402

pytestmark = pytest.mark.gpu
FAR = (1 << 31) + 4096  # bytes: the third row starts above 2^32
F32, BF16 = 0, 1


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


def done(status):
    assert status == 1


def spread(x, pitch):
    """x's rows of bytes, `pitch` apart."""
    raw = x.contiguous().view(len(x), -1).view(torch.uint8)
    buf = torch.empty((len(x) - 1) * pitch + raw.shape[1], dtype=torch.uint8, device="cuda")
    for i, row in enumerate(raw):
        buf[i * pitch:i * pitch + len(row)] = row
    return buf


def norm(x, dy, image, pixel, n, p, c, g):
    dev = dict(device="cuda")
    y, dx = (torch.empty(n, p, c, dtype=torch.bfloat16, **dev) for _ in range(2))
    mean, rstd = torch.empty(n, g, **dev), torch.empty(n, g, **dev)
    dgamma, dbeta = torch.empty(c, **dev), torch.empty(c, **dev)
    gamma, beta = torch.linspace(0.5, 1.5, c, **dev), torch.linspace(-1, 1, c, **dev)
    ws = torch.empty(layers.group_norm_workspace_bytes(n, p, c, g, BF16, True),
                     dtype=torch.uint8, **dev)
    done(layers.group_norm_device(x, image, pixel, gamma, beta, y, mean, rstd, ws, n, p, c, g,
                                  1e-5, 1, BF16))
    done(layers.group_norm_backward_device(x, image, pixel, dy, image, pixel, gamma, beta, mean,
                                           rstd, dx, dgamma, dbeta, ws, n, p, c, g, 1, BF16))
    torch.cuda.synchronize()
    return y, mean, rstd, dx, dgamma, dbeta


@pytest.mark.parametrize("p", [64, 30000])
def test_images_far_apart(p):
    n, c, g = 3, 32, 4
    x, dy = (torch.randn(n, p, c, device="cuda").bfloat16() for _ in range(2))
    near = norm(x, dy, p * c * 2, c * 2, n, p, c, g)
    far = norm(spread(x, FAR), spread(dy, FAR), FAR, c * 2, n, p, c, g)
    for a, b in zip(near, far):
        assert torch.equal(a, b)


def test_pixels_far_apart():
    p, c, g = 3, 64, 2
    x, dy = (torch.randn(1, p, c, device="cuda").bfloat16() for _ in range(2))
    near = norm(x, dy, p * c * 2, c * 2, 1, p, c, g)
    far = norm(spread(x[0], FAR), spread(dy[0], FAR), 0, FAR, 1, p, c, g)
    for a, b in zip(near, far):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n,k", [(8, 2), (64, 4), (1000, 8)])
def test_logits_far_apart(n, k):
    x = torch.randn(3, n, device="cuda")

    def both(logits, stride):
        e, w = (torch.empty(3, k, dtype=d, device="cuda") for d in (torch.int32, torch.float32))
        dl = torch.empty(3, n, device="cuda")
        done(layers.route_device(logits, stride, None, None, e, w, 3, n, k, 1, 1, 0, False, 1.0,
                                 F32))
        done(layers.route_backward_device(logits, stride, e, w, dl, 3, n, k, 0, False, 1.0, F32))
        torch.cuda.synchronize()
        return e, w, dl

    for a, b in zip(both(x, n * 4), both(spread(x, FAR), FAR)):
        assert torch.equal(a, b)


def integers(rows, k):
    """Codes and scales of rows of -3 .. 3, which quantise exactly."""
    x = torch.randint(-3, 4, (rows, k), device="cuda").float()
    return x, quantised(x, k * 4, rows, k)


def quantised(x, stride, rows, k):
    kp = layers.mx4_padded(k)
    codes = torch.empty(rows, kp // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, kp // 32, dtype=torch.uint8, device="cuda")
    done(layers.mx4_quantise_device(x, stride, codes, scales, rows, k, F32))
    return codes, scales


@pytest.mark.parametrize("k", [100, 256])
def test_quantised_rows_far_apart(k):
    x = torch.randn(3, k, device="cuda")
    for a, b in zip(quantised(x, k * 4, 3, k), quantised(spread(x, FAR), FAR, 3, k)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m", [5, 40, 700])
def test_gathered_rows_above_4_gib(m):
    """The staged tiles reach 4 GiB from the first row: such a product goes to
    the few-row kernel."""
    k, n, rows = 2048, 512, (1 << 22) + 1000
    x, (codes, scales) = integers(m, k)
    w, (w_codes, w_scales) = integers(n, k)
    big = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
    big_scales = torch.empty(rows, k // 32, dtype=torch.uint8, device="cuda")
    at = torch.cat([torch.arange(m - m // 2), rows - 1 - torch.arange(m // 2)]).cuda()
    big[at], big_scales[at] = codes, scales
    out = torch.empty(m, n, device="cuda")
    done(layers.mx4_product_device(big, big_scales, rows, at.int(), w_codes, w_scales, None, None,
                                   None, out, m, n, k, 1, 0, F32))
    torch.cuda.synchronize()
    assert torch.equal(out, x @ w.t())


@pytest.mark.parametrize("m", [6, 900])
def test_weights_and_output_above_4_gib(m):
    k, n, experts = 2048, 1500000, 3
    w_codes = torch.randint(0, 256, (experts * n, k // 2), dtype=torch.uint8, device="cuda")
    w_scales = torch.full((experts * n, k // 32), 127, dtype=torch.uint8, device="cuda")
    x, (codes, scales) = integers(m, k)
    offsets = torch.arange(experts + 1, device="cuda", dtype=torch.int32) * (m // experts)
    out = torch.full((m, n), 0.25, device="cuda")
    done(layers.mx4_product_device(codes, scales, m, None, w_codes, w_scales, offsets, None, None,
                                   out, m, n, k, experts, 0, F32))
    torch.cuda.synchronize()
    assert m < 900 or out.numel() * 4 > 1 << 32
    for e in range(experts):
        rows = slice(e * m // experts, (e + 1) * m // experts)
        for first in (0, 700001, n - 300):
            w = torch.empty(300, k, device="cuda")
            done(layers.mx4_values_device(w_codes[e * n + first:], w_scales[e * n + first:], w,
                                          300, k, F32))
            # Multiples of a half below 2^16.
            assert torch.equal(out[rows, first:first + 300], x[rows] @ w.t())
