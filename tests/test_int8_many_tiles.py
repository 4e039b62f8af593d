"""8-bit products of more tiles than one dimension of a grid takes (2^32
threads): the grids, without a GPU, and the results.  Scales are 1 and sums
below 2^24: exact."""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

from . import launches

F32 = layers.DTYPES["f32"]
WIDE, HIGH = 1 << 25, 2 ** 31 - 1


def codes(g, rows, kp):
    return torch.randint(-127, 128, (rows, kp), device="cuda", generator=g, dtype=torch.int8)


@pytest.mark.parametrize("m,n,k,rows,offsets,tiles", [
    (1, WIDE, 128, None, 4096, 4 * (WIDE // 16)),
    (1, WIDE + 17, 128, None, 4096, 4 * (WIDE // 16 + 2)),
    (HIGH, 1, 256, 4096, None, 1 << 27)])
def test_grids(tmp_path_factory, m, n, k, rows, offsets, tiles):
    """Rows of 2^22 workgroups, the last of which may be filled in part."""
    with launches.noted(launches.load(tmp_path_factory.mktemp("names"))) as run:
        (launch,) = run("int8_product_device", a_codes=4096, a_scales=4096,
                        a_rows=50 if rows else m, rows=rows, w_codes=4096, w_scales=4096,
                        offsets=offsets, bias=None, row_scale=None, out=4096, m=m, n=n, k=k,
                        experts=1, act=0, dtype=F32)
    assert launch.name == "few_kernel f32 0" and launch.block == (512, 1, 1)
    assert launch.grid == (1 << 22, -(-tiles // (1 << 22)), 1)
    assert launch.grid[0] * 512 < 2 ** 32


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 17])
def test_more_tiles_than_a_grid_row(torch_cuda, extra):
    """4 runs of rows times 2^21 tiles of 16 columns, 512 threads each."""
    n, k, part = WIDE + extra, 128, 1 << 22
    g = torch.Generator("cuda").manual_seed(extra)
    a, w = codes(g, 1, k), codes(g, n, k)
    one, scales = torch.ones(1, device="cuda"), torch.ones(n, device="cuda")
    offsets = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    out = torch.full((n + 64,), 0.25, device="cuda")
    assert layers.int8_product_device(a, one, 1, None, w, scales, offsets, None, None, out, 1, n,
                                      k, 1, 0, F32, torch.cuda.current_stream()) == 1
    for first in range(0, n, part):
        rows = w[first:first + part]
        # Whole numbers below 2^24: exact in any order.
        assert torch.equal(out[first:first + len(rows)], (rows * a.float()).sum(dim=1)), first
    assert (out[n:] == 0.25).all()


@pytest.mark.gpu
def test_more_rows_than_a_grid_of_staged_tiles(torch_cuda):
    """One column and 2^31 - 1 gathered rows: 2^27 tiles of 16 rows."""
    m, k, a_rows = HIGH, 256, 50
    g = torch.Generator("cuda").manual_seed(5)
    a, w = codes(g, a_rows, k), codes(g, 1, k)
    one = torch.ones(a_rows, device="cuda")
    part = 50 << 20
    some = torch.arange(a_rows, dtype=torch.int32, device="cuda").repeat(part // a_rows)
    rows = torch.empty(m, dtype=torch.int32, device="cuda")
    for first in range(0, m, part):
        rows[first:first + part] = some[:min(part, m - first)]
    out = torch.full((m + 64,), 0.25, device="cuda")
    assert layers.int8_product_device(a, one, a_rows, rows, w, one, None, None, None, out, m, 1, k,
                                      1, 0, F32, torch.cuda.current_stream()) == 1
    want = (a.float() * w.float()).sum(dim=1)[some.long()]
    for first in range(0, m, part):
        size = min(part, m - first)
        assert torch.equal(out[first:first + size], want[:size]), first
    assert (out[m:] == 0.25).all()
    del rows, out
    torch.cuda.empty_cache()
