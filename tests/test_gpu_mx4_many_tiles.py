"""Products of more tiles than one dimension of a grid takes (2^32 threads).
The factors are small integers and multiples of a half, whose sums are exact in
32 bits in any order."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from turbinator_c_amd import layers  # noqa: E402

F32 = layers.DTYPES["f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 17])
def test_more_tiles_than_a_grid_row(torch_cuda, extra):
    """4 runs of rows times 2^21 tiles of 16 columns, 512 threads each."""
    n, k, part = (1 << 25) + extra, 128, 1 << 22
    stream = torch.cuda.current_stream()
    g = torch.Generator("cuda").manual_seed(extra)
    x = torch.randint(-3, 4, (1, k), device="cuda", generator=g).float()
    codes = torch.empty(1, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(1, k // 32, dtype=torch.uint8, device="cuda")
    assert layers.mx4_quantise_device(x, k * 4, codes, scales, 1, k, F32, stream) == 1
    w_codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    w_scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    offsets = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    out = torch.full((n,), 0.25, device="cuda")
    assert layers.mx4_product_device(codes, scales, 1, None, w_codes, w_scales, offsets, None,
                                     None, out, 1, n, k, 1, 0, F32, stream) == 1
    w = torch.empty(part, k, device="cuda")
    for first in range(0, n, part):
        rows = min(part, n - first)
        assert layers.mx4_values_device(w_codes[first:], w_scales[first:], w, rows, k, F32,
                                        stream) == 1
        assert torch.equal(out[first:first + rows], (w[:rows] * x).sum(dim=1)), first


@pytest.mark.gpu
def test_more_rows_than_a_grid_of_staged_tiles(torch_cuda):
    """One column and 2^31 - 1 gathered rows: 2^24 tiles of 128 rows, 256
    threads each."""
    m, k, a_rows = 2 ** 31 - 1, 256, 50
    stream = torch.cuda.current_stream()
    g = torch.Generator("cuda").manual_seed(5)
    a, w = (torch.randint(-3, 4, (r, k), device="cuda", generator=g).float() for r in (a_rows, 1))
    four = []
    for x in (a, w):
        codes = torch.empty(len(x), k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(len(x), k // 32, dtype=torch.uint8, device="cuda")
        assert layers.mx4_quantise_device(x, k * 4, codes, scales, len(x), k, F32, stream) == 1
        four += [codes, scales]
    part = 50 << 20
    some = torch.arange(a_rows, dtype=torch.int32, device="cuda").repeat(part // a_rows)
    rows = torch.empty(m, dtype=torch.int32, device="cuda")
    for first in range(0, m, part):
        rows[first:first + part] = some[:min(part, m - first)]
    out = torch.full((m,), 0.25, device="cuda")
    assert layers.mx4_product_device(*four[:2], a_rows, rows, *four[2:], None, None, None, out, m,
                                     1, k, 1, 0, F32, stream) == 1
    want = (a * w).sum(dim=1)[some.long()]
    for first in range(0, m, part):
        assert torch.equal(out[first:first + part], want[:min(part, m - first)]), first
    del rows, out
    torch.cuda.empty_cache()


def test_outputs_beyond_any_memory_are_refused():
    """More than 2^38 values; before any HIP call."""
    at = 4096
    assert layers.mx4_product_device(at, at, 1 << 20, None, at, at, None, None, None, at, 1 << 20,
                                     (1 << 18) + 1, 16, 1, 0, F32) == 0
