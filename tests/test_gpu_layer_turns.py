"""The layer entries with more work than their grids have workgroups (2^20):
workgroups come round again, over LDS and registers that held another item.
Every result is compared, bit for bit, with calls that need no second turn.
Inputs overlap (strides below a row), so that they stay small."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers  # noqa: E402

pytestmark = pytest.mark.gpu
TURN = 1 << 20
F32, BF16 = layers.DTYPES["f32"], layers.DTYPES["bf16"]


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


def done(status):
    assert status == 1


def norm(x, image, pixel, n, p, c, g, dtype, backward=False):
    """y, mean, rstd, and with `backward` dx, dgamma and dbeta for dy = x."""
    kind = {F32: torch.float32, BF16: torch.bfloat16}[dtype]
    gamma, beta = (torch.linspace(a, a + 1, c, device="cuda") for a in (0.5, -0.5))
    y = torch.empty(n, p, c, dtype=kind, device="cuda")
    mean, rstd = (torch.empty(n, g, device="cuda") for _ in range(2))
    ws = torch.empty(layers.group_norm_workspace_bytes(n, p, c, g, dtype, backward),
                     dtype=torch.uint8, device="cuda")
    if not backward:
        done(layers.group_norm_device(x, image, pixel, gamma, beta, y, mean, rstd, ws, n, p, c, g,
                                      1e-5, 1, dtype))
        return y, mean, rstd
    mean.fill_(0.1)
    rstd.fill_(0.9)
    dgamma, dbeta = (torch.empty(c, device="cuda") for _ in range(2))
    done(layers.group_norm_backward_device(x, image, pixel, x, image, pixel, gamma, beta, mean,
                                           rstd, y, dgamma, dbeta, ws, n, p, c, g, 1, dtype))
    return y, dgamma, dbeta


@pytest.mark.parametrize("c,g", [(8, 2), (12, 4), (8, 8)])
def test_planes_that_a_workgroup_holds(torch_cuda, c, g):
    n = TURN + 70_001
    x = torch.randn(n, 1, c, device="cuda", generator=torch.Generator("cuda").manual_seed(c))
    whole = norm(x, c * 4, c * 4, n, 1, c, g, F32)
    half = n // 2
    for part in (slice(0, half), slice(half, n)):
        some = norm(x[part], c * 4, c * 4, len(x[part]), 1, c, g, F32)
        for a, b in zip(whole, some):
            assert torch.equal(a[part], b)


@pytest.mark.parametrize("backward", [False, True])
def test_planes_in_chunks(torch_cuda, backward):
    """Single elements, 2 bytes from a word's start: chunks of 4,096 pixels."""
    n, p = TURN + 1001, 4000
    buf = torch.randn(n + p + 1, device="cuda",
                      generator=torch.Generator("cuda").manual_seed(2)).bfloat16()
    x = buf[1:]
    assert x.data_ptr() % 4 == 2
    whole = norm(x, 2, 2, n, p, 1, 1, BF16, backward)
    first = TURN - 300
    some = norm(x[first:], 2, 2, n - first, p, 1, 1, BF16, backward)
    assert torch.equal(whole[0][first:], some[0])
    if backward:
        # Terms of about 1 in magnitude.  1,048,576 rows are summed by 128 x 32
        # threads, 256 in sequence, and a few dozen before and after: 2^-15.
        sums = [torch.zeros(1, dtype=torch.float64, device="cuda") for _ in range(2)]
        for i in range(0, n, TURN // 2):
            part = norm(x[i:], 2, 2, min(TURN // 2, n - i), p, 1, 1, BF16, True)
            for s, v in zip(sums, part[1:]):
                s += v.double()
            del part
        for got, want in zip(whole[1:], sums):
            assert ((got.double() - want).abs() <= 2.0 ** -15 * n * p).all()
    else:
        for a, b in zip(whole[1:], some[1:]):
            assert torch.equal(a[first:], b)


def route(x, stride, t, n, k, bias, groups, kept, dtype):
    e = torch.empty(t, k, dtype=torch.int32, device="cuda")
    w = torch.empty(t, k, device="cuda")
    done(layers.route_device(x, stride, bias, None, e, w, t, n, k, groups, kept, 1, True, 1.0,
                             dtype))
    return e, w


@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3), (3, 2)])
@pytest.mark.parametrize("step", [2, 8])
def test_tokens(torch_cuda, groups, kept, step):
    """Four tokens to a workgroup; rows of 16-bit logits `step` apart."""
    n, k, t = 1023 if groups == 3 else 1024, 5, 4 * TURN + 30_001
    logits = torch.randn(t * step + n, device="cuda",
                         generator=torch.Generator("cuda").manual_seed(step)).bfloat16()
    bias = torch.linspace(0, 0.1, n, device="cuda")
    first = 4 * TURN - 2000
    whole = route(logits, 2 * step, t, n, k, bias, groups, kept, BF16)
    some = route(logits[first * step:], 2 * step, t - first, n, k, bias, groups, kept, BF16)
    for a, b in zip(whole, some):
        assert torch.equal(a[first:], b)
    if groups > 1:
        return
    e, w = whole
    for score, renorm in ((0, False), (1, True)):
        dl = torch.empty(t, n, dtype=torch.bfloat16, device="cuda")
        done(layers.route_backward_device(logits, 2 * step, e, w, dl, t, n, k, score, renorm, 1.0,
                                          BF16))
        part = torch.empty(t - first, n, dtype=torch.bfloat16, device="cuda")
        done(layers.route_backward_device(logits[first * step:], 2 * step, e[first:], w[first:],
                                          part, t - first, n, k, score, renorm, 1.0, BF16))
        assert torch.equal(dl[first:], part)
        del dl, part


def test_quantised_rows_and_their_values(torch_cuda):
    """16 items of eight values a row, 256 to a workgroup."""
    k, rows = 128, 16 * TURN + 3001
    x = torch.randn(rows + k, device="cuda",
                    generator=torch.Generator("cuda").manual_seed(4)).bfloat16()

    def quantised(x, rows):
        codes = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(rows, k // 32, dtype=torch.uint8, device="cuda")
        done(layers.mx4_quantise_device(x, 2, codes, scales, rows, k, BF16))
        return codes, scales

    def values(codes, scales):
        out = torch.empty(len(codes), k, dtype=torch.bfloat16, device="cuda")
        done(layers.mx4_values_device(codes, scales, out, len(codes), k, BF16))
        return out

    first = 16 * TURN - 2000
    whole, some = quantised(x, rows), quantised(x[first:], rows - first)
    for a, b in zip(whole, some):
        assert torch.equal(a[first:], b)
    assert torch.equal(values(*whole)[first:], values(*some))
