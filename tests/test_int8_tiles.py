"""8-bit products in each of their tiles (hip_layers.h): that the sizes below
reach the tiles they are listed for, without a GPU (csrc/hip_names.c notes the
kernels that are launched), and on the GPU against whole-number sums: dense and
per expert, gathered rows and rows outside, rows of results on and off 64 bytes,
one to six slices of k (128 values), all types.

Tolerance of a product, u = 2^-24.  The sum is exact; its rounding to 32 bits,
the first scale and the fused second one with the bias cost u each: z is within
3 u (|sum| s_a s_w + |bias|).  The activation's slope is at most 1.13 and its
own error 16 + 2 z^2 units; the row scale adds one, the output its rounding.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

from . import launches
from .test_gpu_int8 import HALF, LEAST, TYPES, U, act64, choices, factors, now

TILES = {"tile_kernel 2 2 2 2 4": "64x64", "tile_kernel 2 2 2 4 3": "64x128",
         "tile_kernel 2 2 4 4 2": "128x128", "tile_kernel 2 4 6 4 2": "192x256",
         "tile_kernel 2 4 8 4 2": "256x256", "few_kernel": "few"}
# tile, m, n, k, experts
CASES = [("few", 40, 64, 128, 1), ("few", 100, 77, 2000, 1), ("few", 60, 64, 500, 5),
         ("64x64", 1119, 350, 128, 1), ("64x64", 445, 448, 250, 1), ("64x64", 302, 437, 500, 1),
         ("64x64", 333, 576, 380, 5), ("64x64", 486, 247, 700, 5),
         ("64x128", 6362, 273, 128, 1), ("64x128", 415, 2368, 256, 1),
         ("64x128", 204, 4188, 700, 1), ("64x128", 8095, 192, 100, 5),
         ("64x128", 456, 1792, 380, 5), ("64x128", 641, 1225, 500, 5),
         ("128x128", 8752, 403, 100, 1), ("128x128", 8500, 448, 250, 1),
         ("128x128", 5735, 642, 700, 1), ("128x128", 1526, 2496, 380, 5),
         ("128x128", 6599, 524, 250, 5),
         ("192x256", 8229, 916, 100, 1), ("192x256", 6584, 1216, 256, 1),
         ("192x256", 8349, 926, 700, 1), ("192x256", 2497, 3136, 380, 5),
         ("192x256", 6435, 1159, 250, 5),
         ("256x256", 4612, 2561, 100, 1), ("256x256", 4626, 2624, 256, 1),
         ("256x256", 6961, 1693, 700, 1), ("256x256", 4100, 2752, 380, 5),
         ("256x256", 3083, 3641, 380, 5), ("256x256", 2904, 3904, 700, 5)]
# n, and rows of the same matrix that go through each of the tiles (k 300).
SHARED = [(2048, {"few": 20, "64x64": 300, "64x128": 900, "128x128": 3000, "192x256": 5000,
                  "256x256": 7000}),
          (1700, {"few": 20, "64x64": 300, "64x128": 1375, "128x128": 3475, "192x256": 5800,
                  "256x256": 7950})]
SHARED_K = 300


@pytest.fixture(scope="module")
def noted(tmp_path_factory):
    with launches.noted(launches.load(tmp_path_factory.mktemp("names"))) as run:
        yield run


def tile_of(noted, m, n, k, experts=1, dtype="f32", rows=None, act="none"):
    at = 4096
    (launch,) = noted("int8_product_device", a_codes=at, a_scales=at, a_rows=m, rows=rows,
                      w_codes=at, w_scales=at, offsets=at if experts > 1 else None, bias=None,
                      row_scale=None, out=at, m=m, n=n, k=k, experts=experts,
                      act=layers.ACTS[act], dtype=layers.DTYPES[dtype])
    words = launch.name.split()
    assert words[1] == dtype and words[2] == str(layers.ACTS[act])
    return TILES[" ".join(words[:1] + words[3:])]


@pytest.mark.parametrize("tile,m,n,k,experts", CASES)
def test_cases_reach_their_tiles(noted, tile, m, n, k, experts):
    for dtype in ("f32", "bf16", "f16"):
        for rows in (None, 4096):
            assert tile_of(noted, m, n, k, experts, dtype, rows, "gelu") == tile


def test_every_tile_has_its_cases(noted):
    """Dense and per expert, on and off 64 bytes, and for the staged tiles one
    slice, two and more than their buffers."""
    for tile in TILES.values():
        mine = [c[1:] for c in CASES if c[0] == tile]
        assert {e > 1 for *_, e in mine} == {False, True}, tile
        assert {n % 32 == 0 for _, n, _, _ in mine} == {False, True}, tile
        if tile != "few":
            slices = {-(-k // 128) for _, _, k, _ in mine}
            assert {1, 2} <= slices and max(slices) >= 4, tile
    for n, rows in SHARED:
        assert set(rows) == set(TILES.values())
        for tile, m in rows.items():
            assert tile_of(noted, m, n, SHARED_K) == tile


def launch_product(a, sa, w, sw, rows, offsets, bias, row_scale, m, n, k, experts, act, dtype,
                   shift=0):
    buffer = torch.full((shift + m * n + 64,), 7.0, dtype=dtype, device="cuda")
    out = buffer[shift:]
    assert layers.int8_product_device(a, sa, len(a), rows, w, sw, offsets, bias, row_scale, out,
                                      m, n, k, experts, layers.ACTS[act], layers.DTYPES[dtype],
                                      now()) == 1
    torch.cuda.synchronize()
    assert (buffer[shift + m * n:] == 7).all() and (buffer[:shift] == 7).all()
    return out[:m * n].view(m, n)


def check(m, n, k, experts, dtype, act, bias, rows=None, a_rows=None, offsets=None,
          row_scale=False, shift=0):
    """As the entry's own test, with the sums in 64 bits on the GPU (whole
    numbers below 2^53: exact)."""
    g = torch.Generator().manual_seed(m + 3 * n + 7 * k)
    a, sa = (v.cuda() for v in factors(g, a_rows or m, k))
    w, sw = (v.cuda() for v in factors(g, experts * n, k))
    b = torch.randn(experts, n, generator=g).cuda() if bias else None
    scale = torch.rand(m, generator=g).cuda() if row_scale else None
    rows, offsets = (v if v is None else v.cuda() for v in (rows, offsets))
    got = launch_product(a, sa, w, sw, rows, offsets, b, scale, m, n, k, experts, act, dtype,
                         shift)
    at = torch.arange(m, device="cuda") if rows is None else rows.long()
    there = (at >= 0) & (at < len(a))
    expert = torch.zeros(m, dtype=torch.long, device="cuda")
    if offsets is not None:
        r = torch.arange(m, device="cuda")
        expert = (r[:, None] >= offsets.long()[None, :]).sum(1) - 1
        there &= (expert >= 0) & (expert < experts)
    z, size = (torch.zeros(m, n, dtype=torch.float64, device="cuda") for _ in range(2))
    for x in range(experts):
        mine = (there & (expert == x)).nonzero()[:, 0]
        if len(mine):
            s = a[at[mine]].double() @ w[x * n:(x + 1) * n].double().T
            s = s * sa[at[mine]].double()[:, None] * sw[x * n:(x + 1) * n].double()
            z[mine] = s if b is None else s + b[x].double()
            size[mine] = s.abs() if b is None else s.abs() + b[x].double().abs()
    want = act64(z, act)
    bound = 1.13 * 3 * U * size + (16 + 2 * z * z) * U * want.abs()
    if scale is not None:
        want, bound = want * scale.double()[:, None], bound * scale.double()[:, None]
        bound = bound + U * want.abs()
    bound = bound + HALF[dtype] * want.abs() * 1.01 + LEAST[dtype]
    assert ((got.double() - want).abs() <= bound)[there].all()
    assert (got[~there] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile,m,n,k,experts", CASES)
def test_products(torch_cuda, tile, m, n, k, experts, dtype):
    g = torch.Generator().manual_seed(m + n)
    if experts == 1:
        check(m, n, k, 1, dtype, "none", True)
        check(m, n, k, 1, dtype, "gelu", False, row_scale=True, shift=3)
        rows, _ = choices(g, m, 1, m // 2 + 1, 0.05)
        check(m, n, k, 1, dtype, "none", False, rows, m // 2 + 1)
        return
    rows, offsets = choices(g, m, experts, m // 2 + 1, 0.05)
    check(m, n, k, experts, dtype, "silu", True, rows, m // 2 + 1, offsets, True)
    # In order, rows before the first expert's and behind the last one's.
    offsets[0], offsets[-1] = 3, m - 5
    offsets = torch.cummax(offsets, 0).values.clamp(max=m - 5).int()
    check(m, n, k, experts, dtype, "none", False, offsets=offsets, shift=1)
    check(m, n, k, experts, dtype, "none", True, offsets=offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows", SHARED)
def test_a_row_in_every_tile(torch_cuda, n, rows):
    """Sums are exact and the steps behind them the same: a row's results are
    the same bits in all six."""
    g = torch.Generator().manual_seed(n)
    k, most = SHARED_K, max(rows.values())
    a, sa = (v.cuda() for v in factors(g, most, k))
    w, sw = (v.cuda() for v in factors(g, n, k))
    bias, scale = torch.randn(n, generator=g).cuda(), torch.rand(most, generator=g).cuda()
    for dtype in TYPES:
        full = launch_product(a, sa, w, sw, None, None, bias, scale, most, n, k, 1, "gelu", dtype)
        for m in rows.values():
            part = launch_product(a[:m], sa, w, sw, None, None, bias, scale, m, n, k, 1, "gelu",
                                  dtype)
            assert torch.equal(part, full[:m])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,experts", [(3000, 3500, 3500, 1), (4096, 4096, 4096, 1),
                                           (16384, 2048, 1024, 8)])
def test_many_slices(torch_cuda, m, n, k, experts):
    """The largest tiles over long rows, as training batches have them."""
    g = torch.Generator().manual_seed(k)
    rows, offsets = choices(g, m, experts, m // 2 + 1) if experts > 1 else (None, None)
    check(m, n, k, experts, torch.bfloat16, "silu", True, rows, rows is not None and m // 2 + 1,
          offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(5000, 2048), (7000, 2048), (5800, 1700), (7950, 1700)])
def test_nan_scales(torch_cuda, m, n):
    """A NaN scale makes its row or column NaN, and nothing else."""
    g = torch.Generator().manual_seed(1)
    a, sa = (v.cuda() for v in factors(g, m, SHARED_K))
    w, sw = (v.cuda() for v in factors(g, n, SHARED_K))
    bad_rows, bad_columns = torch.tensor([2, 200, m - 1]), torch.tensor([0, 255, n - 1])
    sa[bad_rows.cuda()], sw[bad_columns.cuda()] = float("nan"), float("nan")
    for dtype in TYPES:
        got = launch_product(a, sa, w, sw, None, None, None, None, m, n, SHARED_K, 1, "silu",
                             dtype)
        nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        nan[bad_rows.cuda()] = True
        nan[:, bad_columns.cuda()] = True
        assert torch.equal(got.isnan(), nan)
