"""Products per expert large enough for the staged tiles (hip_layers.h): rows
gathered and in order, rows from nowhere, rows before the first expert and
behind the last, widths of an odd number of steps of 128, every type, NaN
blocks.  The tolerances are those of the products in test_gpu_mx4.py."""
from __future__ import annotations

import math

import pytest
import torch

from turbinator_c_amd import layers

from .test_gpu_mx4 import check_product, operands, product, quantise

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def bounds_of(before, counts):
    at = [before]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


# Above 2^18 outputs and 32 rows an expert on average: tiles of 128 for the
# first ones, of 256 for the last (two rounds of 128-tiles, one of 256).
SIZES = [((130, 1, 0, 257, 16), 701, 256), ((130, 1, 0, 257, 16), 1000, 384),
         ((0, 0, 700, 0), 512, 640), ((64, 64, 64), 2000, 1000),
         ((900, 0, 1700, 5, 1650), 2304, 200), ((900, 0, 1700, 5, 1650), 2306, 384)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("counts,n,k", SIZES, ids=str)
def test_staged_experts(torch_cuda, counts, n, k, dtype):
    experts, a_rows = len(counts), 90
    for before, behind in ((0, 0), (2, 70)):
        m = before + sum(counts) + behind
        offsets = bounds_of(before, counts)
        g = torch.Generator().manual_seed(m)
        rows = torch.randint(0, a_rows, (m,), generator=g).to(torch.int32).cuda()
        rows[::9] = -1
        rows[5::11] = a_rows
        print(counts, n, k, before, dtype, flush=True)
        check_product(n, m, n, k, dtype, ["silu", "gelu"][before // 2], True, experts, offsets,
                      rows, a_rows, True)
        check_product(n, m, n, k, dtype, "none", False, experts, offsets)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
def test_staged_epilogues(torch_cuda, name, dtype):
    for with_bias in (False, True):
        for with_scale in (False, True):
            check_product(9, 300, 1100, 384, dtype, name, with_bias, with_scale=with_scale)


def test_staged_offsets_out_of_range(torch_cuda):
    offsets = torch.tensor([-5, 100, 1000, 2000], dtype=torch.int32, device="cuda")
    check_product(3, 400, 700, 384, torch.float32, "none", True, 3, offsets)
    a, w = operands(1, 400, 700, 384, 3)
    for bad in ([300, 100, 350, 0], [400, 0, 400, 0], [70, 70, 30, 900]):
        product(a, 400, None, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), None, None,
                400, 700, 384, 3, "none", torch.float32)


@pytest.mark.parametrize("k", [256, 384, 640, 1000])
@pytest.mark.parametrize("at", [0, 100, 130, -1])
def test_staged_nan_stays_in_its_rows_and_column(torch_cuda, k, at):
    """One NaN among the rows of A, gathered several times, and an Inf in a
    column of one expert."""
    counts, n, a_rows = (300, 150, 260), 701, 64
    m, experts = sum(counts), len(counts)
    a, w = (torch.randn((r, k), generator=torch.Generator().manual_seed(r)).cuda()
            for r in (a_rows, experts * n))
    a[7, at] = float("nan")
    w[n + 33, at] = math.inf
    rows = (torch.arange(m, device="cuda") % a_rows).int()
    offsets = bounds_of(0, counts)
    out = product(quantise(a), a_rows, rows, quantise(w), offsets, None, None, m, n, k, experts,
                  "none", torch.float32)
    bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    bad[rows == 7] = True
    bad[300:450, 33] = True
    assert torch.equal(torch.isnan(out), bad)


def test_staged_other_stream(torch_cuda):
    counts, n, k, a_rows = (900, 0, 1700, 5, 1650), 2304, 256, 700
    m, experts = sum(counts), len(counts)
    a, w = operands(5, a_rows, n, k, experts)
    rows = (torch.arange(m, device="cuda") * 7 % a_rows).int()
    offsets = bounds_of(0, counts)
    torch.cuda.synchronize()
    first, second = (product(a, a_rows, rows, w, offsets, None, None, m, n, k, experts, "silu",
                             torch.bfloat16, s) for s in (None, torch.cuda.Stream()))
    assert torch.equal(first, second)
