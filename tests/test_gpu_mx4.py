"""Microscaled 4-bit floating point (hip_layers.h): codes and scales bit for
bit against a plain quantiser (every tie and its neighbours, subnormals, NaN
and Inf, zeros, odd widths, strides), the values, and products against 64 bits:
one row to many, odd sizes, experts with and without rows, rows outside.

Tolerance of a product.  Each factor is exact; the matrix instruction sums in
32 bits, its sums of a step off by a few units of the largest magnitude, so a
sum of s steps is within 2^-20 of sum |a w|.  Bias, activation (slope at most
1.13) and row scale add 16 u of their size, the output its rounding.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def plain_quantise(x):
    """codes [rows, kp / 2], scales [rows, kp / 32] of float64 rows, by search."""
    rows, k = x.shape
    kp = -(-k // 128) * 128
    v = np.zeros((rows, kp // 32, 32))
    v.reshape(rows, kp)[:, :k] = x
    top = np.abs(v).max(axis=2)
    bad = ~np.isfinite(v).all(axis=2)
    power = np.frexp(np.where(bad | (top == 0), 1.0, top))[1] - 3
    scale = np.where(top == 0, 0, np.maximum(power + 127, 0))
    scale = np.where(bad, 255, scale)
    u = np.where(bad[..., None], 0.0, np.abs(v)) / np.exp2(np.where(bad, 0, scale - 127.0))[..., None]
    u = np.minimum(u, 6.0)
    # Nearest value; of two at the same distance the one with the even code.
    d = np.abs(u[..., None] - VALUES)
    near = d == d.min(axis=-1, keepdims=True)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[near[..., order].argmax(axis=-1)]
    code = code + 8 * (np.signbit(v) & ~bad[..., None])
    code = code.reshape(rows, kp // 2, 2)
    return (code[..., 0] + 16 * code[..., 1]).astype(np.uint8), scale.astype(np.uint8)


def plain_values(codes, scales, k):
    rows = len(codes)
    code = np.stack([codes & 15, codes >> 4], axis=2).reshape(rows, -1, 32)
    v = np.where(code & 8, -1.0, 1.0) * VALUES[code & 7]
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(float) - 127))
    return (v * unit[..., None]).reshape(rows, -1)[:, :k]


def quantise(x, stream=None):
    m, k = x.shape
    kp = layers.mx4_padded(k)
    codes = torch.full((m * kp // 2 + 16,), 0xa5, dtype=torch.uint8, device="cuda")
    scales = torch.full((m * kp // 32 + 16,), 0xa5, dtype=torch.uint8, device="cuda")
    assert layers.mx4_quantise_device(x, x.stride(0) * x.element_size(), codes, scales, m, k,
                                      layers.DTYPES[x.dtype],
                                      stream or torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (codes[-16:] == 0xa5).all() and (scales[-16:] == 0xa5).all()
    return codes[:-16].view(m, kp // 2), scales[:-16].view(m, kp // 32)


def values(codes, scales, k, dtype):
    out = torch.full((len(codes) * k + 16,), 7.0, dtype=dtype, device="cuda")
    assert layers.mx4_values_device(codes, scales, out, len(codes), k, layers.DTYPES[dtype],
                                    torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (out[-16:] == 7).all()
    return out[:-16].view(len(codes), k)


def check_quantise(x):
    codes, scales = quantise(x)
    want_c, want_s = plain_quantise(x.double().cpu().numpy())
    assert (scales.cpu().numpy() == want_s).all()
    assert (codes.cpu().numpy() == want_c).all()
    k = x.shape[1]
    want = torch.from_numpy(plain_values(want_c, want_s, k))
    for dtype in TYPES:
        assert torch.equal(torch.nan_to_num(values(codes, scales, k, dtype).cpu(), nan=9e3),
                           torch.nan_to_num(want.to(torch.float32).to(dtype), nan=9e3))
    return codes, scales


def rows_of(seed, m, k, dtype, pitch=None):
    g = torch.Generator().manual_seed(seed)
    pitch = pitch or k
    wide = torch.full((m, pitch), float("nan"))
    size = torch.exp2(6 * torch.randn((m, -(-k // 32)), generator=g)).repeat_interleave(32, 1)
    wide[:, pitch - k:] = torch.randn((m, k), generator=g) * size[:, :k]
    if dtype == torch.float16:
        wide = wide.clamp(-6e4, 6e4)
    return wide.to(dtype).cuda()[:, pitch - k:]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 127), (2, 128), (7, 129),
                                 (33, 500), (4, 2000), (300, 64), (1, 8192)])
def test_quantise(torch_cuda, m, k, dtype):
    check_quantise(rows_of(m + k, m, k, dtype))
    for pitch in (k + 1, k + 8):
        check_quantise(rows_of(m + k, m, k, dtype, pitch))


def test_ties_and_their_neighbours(torch_cuda):
    """Every midpoint and value times a scale, the floats next to them, both
    signs; the block's scale set by 4 (and by values that saturate)."""
    mids = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7],
                    np.float32)
    around = np.concatenate([mids, np.nextafter(mids, np.float32(9)),
                             np.nextafter(mids, np.float32(-9))])
    around = np.concatenate([around, -around])
    around[np.abs(around) >= 8] = 0
    rows = []
    for scale in (2.0 ** -126, 2.0 ** -100, 1.0, 2.0 ** 60, 2.0 ** 125):
        for i in range(0, len(around), 31):
            block = np.zeros(32, np.float32)
            block[:len(around[i:i + 31])] = around[i:i + 31]
            block[31] = 4
            rows.append(block * np.float32(scale))
    check_quantise(torch.from_numpy(np.array(rows, np.float32)).cuda())


def test_special_blocks(torch_cuda):
    x = torch.randn((12, 96), generator=torch.Generator().manual_seed(3))
    x[0] = 0
    x[1] = -0.0
    x[2, 40] = float("nan")
    x[3, 40] = math.inf
    x[4, 95] = -math.inf
    x[5] *= 1e-40                       # subnormals
    x[6] = torch.finfo(torch.float32).tiny
    x[7] = 1.4e-45
    x[8] = torch.finfo(torch.float32).max
    x[9, ::2] = torch.finfo(torch.float32).max
    x[10, 5] = 2.0 ** -125              # the last scale before the lowest
    x[10, 6:] = 0
    codes, scales = check_quantise(x.cuda())
    assert scales[2, 1] == 255 and scales[2, 0] != 255 and (codes[2, 16:32] == 0).all()


def test_padding_is_zero(torch_cuda):
    codes, scales = quantise(rows_of(1, 9, 40, torch.float32))
    assert (codes[:, 20:] == 0).all() and (scales[:, 2:] == 0).all()


# --------------------------------------------------------------------------
# Products


def act(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    return torch.nn.functional.gelu(z) if name == "gelu" else z


def operands(seed, m, n, k, experts):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn((m, k), generator=g) * torch.exp2(2 * torch.randn((m, 1), generator=g))
    w = torch.randn((experts * n, k), generator=g) / math.sqrt(k)
    return quantise(a.cuda()), quantise(w.cuda())


def product(a, a_rows, rows, w, offsets, bias, row_scale, m, n, k, experts, name, dtype,
            stream=None):
    out = torch.full((m * n + 16,), 7.0, dtype=dtype, device="cuda")
    assert layers.mx4_product_device(*a, a_rows, rows, *w, offsets, bias, row_scale, out, m, n,
                                     k, experts, layers.ACTS[name], layers.DTYPES[dtype],
                                     stream or torch.cuda.current_stream()) == 1
    torch.cuda.synchronize()
    assert (out[-16:] == 7).all()
    return out[:-16].view(m, n)


def check_product(seed, m, n, k, dtype, name="none", with_bias=True, experts=1, offsets=None,
                  rows=None, a_rows=None, with_scale=False):
    a_rows = a_rows or m
    a, w = operands(seed, a_rows, n, k, experts)
    g = torch.Generator().manual_seed(seed + 1)
    bias = (torch.randn((experts, n), generator=g)).cuda() if with_bias else None
    row_scale = torch.rand(m, generator=g).cuda() if with_scale else None
    got = product(a, a_rows, rows, w, offsets, bias, row_scale, m, n, k, experts, name, dtype)
    av, wv = (torch.from_numpy(plain_values(c.cpu().numpy(), s.cpu().numpy(), k)).cuda()
              for c, s in (a, w))
    r = torch.arange(m, device="cuda") if rows is None else rows.long()
    live = (r >= 0) & (r < a_rows)
    av = torch.where(live[:, None], av[r.clamp(0, a_rows - 1)], 0.0)
    bounds = [0, m] if offsets is None else offsets.clamp(0, m).tolist()
    want, size = (torch.zeros((m, n), dtype=torch.float64, device="cuda") for _ in range(2))
    for x in range(experts):
        lo, hi = bounds[x], bounds[x + 1]
        if hi <= lo:
            continue
        we = wv[x * n:(x + 1) * n]
        z = av[lo:hi] @ we.T
        size[lo:hi] = 2.0 ** -20 * (av[lo:hi].abs() @ we.abs().T)
        if with_bias:
            z = z + bias[x].double()
        size[lo:hi] = 1.13 * (size[lo:hi] + 16 * U * (1 + z.abs()))
        y = act(z, name)
        scale = row_scale[lo:hi, None].double() if with_scale else 1.0
        want[lo:hi] = y * scale
        size[lo:hi] *= scale
    used = torch.zeros(m, dtype=torch.bool, device="cuda")
    used[bounds[0]:bounds[-1]] = True
    want[~(live & used)] = 0
    over = (got.double() - want).abs() - size - HALF_ULP[dtype] * want.abs() - LEAST[dtype]
    assert over.max() <= 0, (over.max(), m, n, k)
    assert (got[~(live & used)] == 0).all()
    return got


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 33), (10, 64, 512), (15, 100, 129), (16, 65, 2048),
         (17, 256, 1000), (33, 130, 640), (64, 64, 4096), (65, 1000, 100), (100, 300, 300),
         (129, 127, 1500), (256, 512, 256), (300, 260, 128), (513, 511, 384), (1000, 1024, 1024),
         (10, 4096, 4096), (320, 2048, 2048), (2050, 96, 70)]
# Every shape of the product: few rows with one, two and four row tiles, staged
# tiles of 128 and of 256; widths with one to eight steps of 128; ragged ends.
SIZES += [(m, n, k) for m, n in ((33, 1500), (60, 2100), (200, 9000), (700, 500), (1300, 1111),
                                 (4200, 2200)) for k in (100, 250, 300, 500, 512, 700, 900, 1024)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_product(torch_cuda, size, dtype):
    m, n, k = size
    print(size, dtype, flush=True)
    check_product(m + n, m, n, k, dtype, ["none", "silu", "gelu"][(m + n) % 3], n % 2 == 0)


@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
@pytest.mark.parametrize("m", [4, 40, 400])
def test_epilogues(torch_cuda, m, name):
    for with_bias in (False, True):
        for with_scale in (False, True):
            check_product(m, m, 144, 256, torch.bfloat16, name, with_bias, with_scale=with_scale)


@pytest.mark.parametrize("n,k", [(64, 128), (200, 300), (256, 512)])
@pytest.mark.parametrize("counts", [(3, 0, 5, 1), (64, 64, 64), (0, 0, 700, 0), (1,) * 20,
                                    (130, 1, 0, 257, 16), (0, 0)], ids=str)
def test_experts(torch_cuda, counts, n, k):
    """Experts with none, one and many rows; rows gathered by index, some of
    them from nowhere; rows before the first expert and behind the last."""
    experts, live = len(counts), sum(counts)
    for before, behind in ((0, 0), (2, 70)):
        m = max(1, before + live + behind)
        at = [before]
        for c in counts:
            at.append(at[-1] + c)
        offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
        g = torch.Generator().manual_seed(m)
        rows = torch.randint(0, 50, (m,), generator=g).to(torch.int32).cuda()
        rows[::9] = -1
        rows[5::11] = 50
        print(counts, n, k, before, flush=True)
        check_product(n, m, n, k, torch.bfloat16, "silu", True, experts, offsets, rows, 50, True)
        check_product(n, m, n, k, torch.float32, "none", False, experts, offsets)


def test_offsets_out_of_range(torch_cuda):
    """Offsets below 0 and above m are taken as 0 and m; decreasing ones stay
    inside the output."""
    offsets = torch.tensor([-5, 10, 1000, 2000], dtype=torch.int32, device="cuda")
    check_product(3, 40, 64, 128, torch.float32, "none", True, 3, offsets)
    a, w = operands(1, 40, 64, 128, 3)
    for bad in ([30, 10, 35, 0], [40, 0, 40, 0], [7, 7, 3, 90]):
        product(a, 40, None, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), None, None,
                40, 64, 128, 3, "none", torch.float32)


def test_nan_stays_in_its_row_and_column(torch_cuda):
    a = torch.randn((40, 256), generator=torch.Generator().manual_seed(3)).cuda()
    w = torch.randn((70, 256), generator=torch.Generator().manual_seed(4)).cuda()
    a[7, 100] = float("nan")
    w[33, 200] = math.inf
    out = product(quantise(a), 40, None, quantise(w), None, None, None, 40, 70, 256, 1, "none",
                  torch.float32)
    bad = torch.zeros((40, 70), dtype=torch.bool, device="cuda")
    bad[7], bad[:, 33] = True, True
    assert torch.equal(torch.isnan(out), bad)


def test_other_stream(torch_cuda):
    a, w = operands(5, 300, 256, 512, 1)
    torch.cuda.synchronize()
    first, second = (product(a, 300, None, w, None, None, None, 300, 256, 512, 1, "silu",
                             torch.bfloat16, s) for s in (None, torch.cuda.Stream()))
    assert torch.equal(first, second)


def test_refusals(torch_cuda):
    x = torch.zeros((4, 64), device="cuda")
    codes = torch.full((1024,), 9, dtype=torch.uint8, device="cuda")
    scales = torch.full((1024,), 9, dtype=torch.uint8, device="cuda")
    out = torch.full((1024,), 7.0, device="cuda")
    idx = torch.zeros(16, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream()
    good = [x, 256, codes, scales, 4, 64, 0]
    for i, v in ((0, None), (2, None), (3, None), (4, 0), (4, 2 ** 31), (5, 0), (5, 2 ** 31),
                 (6, 3), (1, 254), (0, x.data_ptr() + 2), (2, codes.data_ptr() + 8),
                 (3, scales.data_ptr() + 2)):
        args = list(good)
        args[i] = v
        assert layers.mx4_quantise_device(*args, stream) == 0, i
    good = [codes, scales, out, 4, 64, 0]
    for i, v in ((0, None), (1, None), (2, None), (3, 0), (4, 0), (5, -1),
                 (0, codes.data_ptr() + 8), (1, scales.data_ptr() + 1),
                 (2, out.data_ptr() + 2)):
        args = list(good)
        args[i] = v
        assert layers.mx4_values_device(*args, stream) == 0, i
    good = [codes, scales, 4, idx, codes, scales, idx, None, None, out, 4, 8, 64, 2, 0, 0]
    for i, v in ((0, None), (1, None), (2, 0), (4, None), (5, None), (9, None), (10, 0),
                 (11, 0), (12, 0), (13, 0), (13, 1025), (14, 3), (14, -1), (15, 3), (6, None),
                 (0, codes.data_ptr() + 8), (1, scales.data_ptr() + 2),
                 (4, codes.data_ptr() + 8), (5, scales.data_ptr() + 2),
                 (9, out.data_ptr() + 2), (10, 2 ** 31), (11, 2 ** 30), (12, 2 ** 31)):
        args = list(good)
        args[i] = v
        assert layers.mx4_product_device(*args, stream) == 0, i
    args = list(good)
    args[3], args[10] = None, 5
    assert layers.mx4_product_device(*args, stream) == 0
    torch.cuda.synchronize()
    assert (codes == 9).all() and (scales == 9).all() and (out == 7).all()
