"""Rows in 8-bit integers (hip_layers.h): codes and scales bit for bit against a
plain quantiser (ties, subnormals, NaN and Inf, zeros, odd widths, strides), the
values, and products against whole-number sums: one row to many, odd sizes,
experts with and without rows, rows outside.

Tolerance of a product, u = 2^-24.  The sum is exact; its rounding to 32 bits,
the first scale and the fused second one with the bias cost u each: z is within
3 u (|sum| s_a s_w + |bias|).  The activation's slope is at most 1.13 and its
own error 16 + 2 z^2 units; the row scale adds one, the output its rounding.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F127, TINY = np.float32(127), np.float32(2.0 ** -126)


def now():
    return torch.cuda.current_stream()


def plain_quantise(x):
    """codes [rows, kp] and scales [rows] of float32 rows, in numpy's 32-bit arithmetic."""
    x = x.float().cpu().numpy()
    rows, k = x.shape
    finite = np.isfinite(x).all(axis=1)
    x = np.where(finite[:, None], x, np.float32(0))
    scale = np.maximum(np.abs(x).max(axis=1) / F127, TINY)
    q = np.rint(x * (np.float32(1) / scale)[:, None])
    assert np.abs(q).max() <= 127
    codes = np.zeros((rows, -(-k // 128) * 128), np.int8)
    codes[:, :k] = q
    return codes, np.where(finite, scale, np.float32(np.nan))


def quantise(x, stream=None):
    m, k = x.shape
    kp = layers.int8_padded(k)
    codes = torch.full((m * kp + 16,), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((m + 4,), 7.0, device="cuda")
    assert layers.int8_quantise_device(x, x.stride(0) * x.element_size(), codes, scales, m, k,
                                       layers.DTYPES[x.dtype], stream or now()) == 1
    torch.cuda.synchronize()
    assert (codes[-16:] == 99).all() and (scales[-4:] == 7).all()
    return codes[:-16].view(m, kp), scales[:-4]


def same(a, b):
    return np.array_equal(np.asarray(a), np.asarray(b), equal_nan=True)


def check_quantise(x):
    codes, scales = quantise(x)
    want_c, want_s = plain_quantise(x)
    assert same(scales.cpu().numpy(), want_s)
    assert same(codes.cpu().numpy(), want_c)
    m, k = x.shape
    with np.errstate(over="ignore"):
        values = torch.from_numpy(want_c[:, :k].astype(np.float32) * want_s[:, None])
    for dtype in TYPES:
        out = torch.full((m * k + 16,), 7.0, dtype=dtype, device="cuda")
        assert layers.int8_values_device(codes, scales, out, m, k, layers.DTYPES[dtype],
                                         now()) == 1
        torch.cuda.synchronize()
        assert (out[-16:] == 7).all()
        assert same(out[:-16].view(m, k).cpu().float().numpy(), values.to(dtype).float().numpy())
    return codes, scales


def rows_of(g, m, k, dtype, pitch=None, shift=0):
    pitch = pitch or k
    wide = torch.full((m * pitch + shift,), float("nan"))
    size = torch.exp2(4 * torch.randn((m, 1), generator=g))
    wide[shift:].view(m, pitch)[:, pitch - k:] = torch.randn((m, k), generator=g) * size
    return wide.to(dtype).cuda()[shift:].view(m, pitch)[:, pitch - k:]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (3, 7), (5, 33), (2, 127), (2, 128), (7, 129),
                                 (33, 500), (6, 2040), (5, 2048), (4, 2049), (3, 2056), (2, 8192),
                                 (2, 8193), (1, 20001), (1000, 64)])
def test_quantise(torch_cuda, m, k, dtype):
    g = torch.Generator().manual_seed(m + k)
    check_quantise(rows_of(g, m, k, dtype))
    check_quantise(rows_of(g, m, k, dtype, k + 1, 1))
    check_quantise(rows_of(g, m, k, dtype, k + 8))


def test_ties_and_their_neighbours(torch_cuda):
    """Every midpoint times a scale that is a power of two, and the floats next
    to it, both signs."""
    mids = np.arange(0, 127, dtype=np.float32) + np.float32(0.5)
    near = np.concatenate([mids, np.nextafter(mids, np.float32(0)),
                           np.nextafter(mids, np.float32(200)), np.arange(128, dtype=np.float32)])
    row = np.concatenate([near, -near, [127.0]]).astype(np.float32)
    for power in (0, -20, 31, -120):
        check_quantise(torch.from_numpy(row[None] * np.float32(2.0 ** power)).cuda())


def test_zeros_subnormals_and_the_largest(torch_cuda):
    x = torch.zeros(9, 40, device="cuda")
    x[1, 3] = -0.0
    x[2, 5] = 1e-45
    x[3] = torch.linspace(-1e-38, 1e-38, 40)
    x[4] = torch.linspace(-127 * 2.0 ** -126, 127 * 2.0 ** -126, 40)
    x[5] = torch.linspace(-3.4e38, 3.4e38, 40)
    x[6, 0] = 3.4028234663852886e38
    x[7] = 1.0
    x[8, 39] = -1e-30
    check_quantise(x)
    check_quantise(x.bfloat16())
    check_quantise(torch.full((2, 9), 65504.0, dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("k", [24, 300, 9000])
def test_rows_that_are_not_finite(torch_cuda, k):
    for dtype in TYPES:
        x = torch.randn(7, k, device="cuda").to(dtype)
        x[1, 0], x[3, k - 1], x[5, k // 2] = float("inf"), float("nan"), -float("inf")
        codes, scales = check_quantise(x)
        assert torch.isnan(scales).cpu().tolist() == [False, True, False, True, False, True, False]


# --------------------------------------------------------------------------


def act64(z, act):
    if act == "silu":
        return torch.nn.functional.silu(z)
    return torch.nn.functional.gelu(z) if act == "gelu" else z


def factors(g, rows, k):
    """Random codes over the whole range, and scales."""
    codes = torch.zeros(rows, layers.int8_padded(k), dtype=torch.int8)
    codes[:, :k] = torch.randint(-127, 128, (rows, k), generator=g).to(torch.int8)
    return codes, torch.exp2(-8 - 2 * torch.rand(rows, generator=g))


def run_product(a, sa, w, sw, rows, offsets, bias, row_scale, m, n, k, experts, act, dtype,
                shift=0):
    buffer = torch.full((shift + m * n + 64,), 7.0, dtype=dtype, device="cuda")
    out = buffer[shift:]
    assert layers.int8_product_device(a, sa, len(a), rows, w, sw, offsets, bias, row_scale, out,
                                      m, n, k, experts, layers.ACTS[act], layers.DTYPES[dtype],
                                      now()) == 1
    torch.cuda.synchronize()
    assert (buffer[-64:] == 7).all() and (buffer[:shift] == 7).all()
    return out[:m * n].view(m, n).cpu()


def check_product(m, n, k, dtype, act="none", bias=True, experts=1, offsets=None, rows=None,
                  a_rows=None, row_scale=False, shift=0, seed=0):
    g = torch.Generator().manual_seed(seed + m + 3 * n + 7 * k)
    a, sa = factors(g, a_rows or m, k)
    w, sw = factors(g, experts * n, k)
    b = torch.randn(experts, n, generator=g) if bias else None
    scale = torch.rand(m, generator=g) if row_scale else None
    cuda = [v if v is None else v.cuda() for v in (a, sa, w, sw, rows, offsets, b, scale)]
    got = run_product(*cuda, m, n, k, experts, act, dtype, shift)
    at = torch.arange(m) if rows is None else rows.long()
    there = (at >= 0) & (at < len(a))
    if offsets is None:
        expert = torch.zeros(m, dtype=torch.long)
    else:
        ends = offsets.long().clamp(0, m)
        r = torch.arange(m)
        expert = (r[:, None] >= ends[None, :]).sum(1) - 1
        there &= (r >= ends[0]) & (r < ends[-1])
    expert = expert.clamp(0, experts - 1)
    z, size = torch.zeros(m, n, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    for x in range(experts):
        mine = (there & (expert == x)).nonzero()[:, 0]
        if not len(mine):
            continue
        # Sums below 2^53: exact in 64-bit floating point.
        s = a[at[mine]].double() @ w[x * n:(x + 1) * n].double().T
        s = s * sa[at[mine]].double()[:, None] * sw[x * n:(x + 1) * n].double()
        z[mine] = s if b is None else s + b[x].double()
        size[mine] = s.abs() if b is None else s.abs() + b[x].double().abs()
    want = act64(z, act)
    bound = 1.13 * 3 * U * size + (16 + 2 * z * z) * U * want.abs()
    if scale is not None:
        want, bound = want * scale.double()[:, None], bound * scale.double()[:, None]
        bound = bound + U * want.abs()
    want = torch.where(there[:, None], want, 0.0)
    bound = torch.where(there[:, None], bound, 0.0) + HALF[dtype] * want.abs() * 1.01
    assert ((got.double() - want).abs() <= bound + LEAST[dtype]).all()
    assert (got[~there] == 0).all()
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 65), (1, 4096, 4096), (2, 5, 128),
                                   (10, 200, 300), (16, 16, 64), (17, 33, 129), (33, 100, 1000),
                                   (64, 512, 512), (100, 77, 2000), (129, 64, 31)])
def test_few_rows(torch_cuda, m, n, k, dtype):
    check_product(m, n, k, dtype)
    check_product(m, n, k, dtype, "silu", False, shift=1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(600, 640, 1), (513, 1024, 64), (600, 700, 128),
                                   (515, 1025, 129), (700, 513, 257), (1000, 999, 384),
                                   (2050, 1030, 640), (4100, 4104, 96)])
def test_many_rows(torch_cuda, m, n, k, dtype):
    check_product(m, n, k, dtype)
    check_product(m, n, k, dtype, "gelu", False, row_scale=True, shift=3)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("m,n,k", [(9, 50, 200), (700, 520, 200)])
def test_activations(torch_cuda, m, n, k, act):
    for dtype in TYPES:
        check_product(m, n, k, dtype, act, row_scale=True)


def choices(g, m, experts, a_rows, missing=0.0):
    """Rows' tokens and the experts' offsets, some experts without any."""
    expert = torch.randint(0, experts, (m,), generator=g)
    expert = torch.where(expert % 3 == 1, 0, expert).sort().values
    offsets = torch.searchsorted(expert, torch.arange(experts + 1)).int()
    rows = torch.randint(0, a_rows, (m,), generator=g)
    rows = torch.where(torch.rand(m, generator=g) < missing,
                       torch.tensor([-1, a_rows, -2 ** 31, 2 ** 31 - 1])
                       [torch.randint(0, 4, (m,), generator=g)], rows)
    return rows.int(), offsets


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k,experts", [(1, 64, 64, 1024), (20, 40, 130, 4), (300, 100, 260, 8),
                                           (1500, 520, 200, 5), (4000, 260, 128, 7),
                                           (5000, 1024, 384, 2), (700, 1000, 65, 70)])
def test_experts(torch_cuda, m, n, k, experts, dtype):
    g = torch.Generator().manual_seed(m)
    rows, offsets = choices(g, m, experts, m // 2 + 1, 0.05)
    check_product(m, n, k, dtype, "silu", True, experts, offsets, rows, m // 2 + 1, True)
    # In order, rows before the first expert's and behind the last one's.
    offsets = offsets.clone()
    offsets[0], offsets[-1] = min(3, m), max(0, m - 5)
    offsets = torch.cummax(offsets, 0).values.clamp(max=max(0, m - 5)).int()
    check_product(m, n, k, dtype, "none", False, experts, offsets)


def test_offsets_past_the_rows(torch_cuda):
    for m, n in ((40, 30), (900, 600)):
        check_product(m, n, 70, torch.float32, experts=2,
                      offsets=torch.tensor([-7, m // 2, 2 ** 31 - 1], dtype=torch.int32))
        check_product(m, n, 70, torch.float32, experts=1,
                      offsets=torch.tensor([0, 0], dtype=torch.int32))


@pytest.mark.parametrize("m,n", [(3, 20), (600, 512)])
def test_largest_sums(torch_cuda, m, n):
    """Codes of 127 all along the longest rows: sums just below 2^31."""
    k = 131072
    a = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    one = torch.ones(max(m, n), device="cuda")
    got = run_product(a, one, w, one, None, None, None, None, m, n, k, 1, "none", torch.float32)
    want = torch.full((m, n), float(127 * 127 * k))
    want[:, 1] = -want[:, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,n", [(5, 40), (700, 600)])
def test_rows_that_are_nan(torch_cuda, m, n):
    """A NaN scale makes its row or column NaN, and nothing else."""
    g = torch.Generator().manual_seed(1)
    a, sa = factors(g, m, 100)
    w, sw = factors(g, n, 100)
    sa[2], sw[7] = float("nan"), float("nan")
    got = run_product(a.cuda(), sa.cuda(), w.cuda(), sw.cuda(), None, None, None, None, m, n, 100,
                      1, "silu", torch.bfloat16)
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[2], nan[:, 7] = True, True
    assert torch.equal(got.isnan(), nan)


def test_same_in_every_shape(torch_cuda):
    """Sums are exact: a row's results do not depend on how many rows go with it."""
    g = torch.Generator().manual_seed(2)
    m, n, k = 1100, 520, 300
    a, sa = (v.cuda() for v in factors(g, m, k))
    w, sw = (v.cuda() for v in factors(g, n, k))
    bias = torch.randn(n, generator=g).cuda()
    for dtype in TYPES:
        full = run_product(a, sa, w, sw, None, None, bias, None, m, n, k, 1, "gelu", dtype)
        for rows in (1, 20, 50, 100, 600):
            part = run_product(a[:rows], sa, w, sw, None, None, bias, None, rows, n, k, 1, "gelu",
                               dtype)
            assert torch.equal(part, full[:rows])


def test_two_streams_and_a_graph(torch_cuda):
    g = torch.Generator().manual_seed(3)
    m, n, k = 700, 640, 1000
    x = rows_of(g, m, k, torch.bfloat16)
    w, sw = (v.cuda() for v in factors(g, n, k))
    codes = torch.empty(m, layers.int8_padded(k), dtype=torch.int8, device="cuda")
    scales, out = torch.empty(m, device="cuda"), torch.empty(m, n, device="cuda").bfloat16()

    def step(stream, codes, scales, out):
        assert layers.int8_quantise_device(x, k * 2, codes, scales, m, k, 1, stream) == 1
        assert layers.int8_product_device(codes, scales, m, None, w, sw, None, None, None, out, m,
                                          n, k, 1, 1, 1, stream) == 1

    step(now(), codes, scales, out)
    torch.cuda.synchronize()
    first = out.clone()
    sides = [torch.cuda.Stream() for _ in range(2)]
    own = [(torch.empty_like(codes), torch.empty_like(scales), torch.empty_like(out))
           for _ in sides]
    torch.cuda.synchronize()
    for _ in range(3):
        for side, buffers in zip(sides, own):
            step(side, *buffers)
    torch.cuda.synchronize()
    assert all(torch.equal(b[2], first) for b in own)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(now(), codes, scales, out)
    for _ in range(3):
        x.copy_(rows_of(g, m, k, torch.bfloat16))
        step(now(), codes, scales, out)
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_past_four_gib(torch_cuda):
    """Gathered rows past 2^32 bytes of codes, in both kinds of kernels."""
    k, a_rows, n = 4096, 1100000, 520
    a = torch.zeros(a_rows, k, dtype=torch.int8, device="cuda")
    assert a.numel() > 2 ** 32
    a[-1] = 2
    a[a_rows - 1000] = 3
    sa = torch.ones(a_rows, device="cuda")
    w = torch.ones(n, k, dtype=torch.int8, device="cuda")
    sw = torch.ones(n, device="cuda")
    for m in (20, 600):
        rows = torch.zeros(m, dtype=torch.int32, device="cuda")
        rows[1], rows[m - 1] = a_rows - 1, a_rows - 1000
        got = run_product(a, sa, w, sw, rows, None, None, None, m, n, k, 1, "none", torch.float32)
        want = torch.zeros(m, n)
        want[1], want[m - 1] = 2 * k, 3 * k
        assert torch.equal(got, want)
