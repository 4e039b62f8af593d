"""The entries for experts' rows, embeddings and 8-bit rows with more work than
their grids have workgroups (2^20), which then take turns: the last turn's rows
against what they must be.  Inputs repeat one row (stride 0) where they can."""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

BF16, F32 = layers.DTYPES["bf16"], layers.DTYPES["f32"]


def now():
    return torch.cuda.current_stream()


def line(width):
    """Whole numbers that bf16 holds."""
    return (torch.arange(width, device="cuda") % 61 - 30).bfloat16()


def all_rows(out, want):
    return all(bool((out[i:i + 16384] == want).all()) for i in range(0, len(out), 16384))


def test_rows_and_sum(torch_cuda):
    """63 pieces a token, 4.4 million in all, four to a workgroup."""
    t, width = 70001, 32000
    x = line(width)
    positions = torch.arange(t, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, t - 1], dtype=torch.int32, device="cuda")
    out = torch.full((t, width), 7.0, dtype=torch.bfloat16, device="cuda")
    assert layers.expert_rows_device(x, 0, offsets, positions, None, out, t, 1, 1, width, BF16,
                                     now()) == 1
    assert all_rows(out[:-1], x) and (out[-1] == 0).all()
    weights = torch.full((t, 1), 2.0, device="cuda")
    assert layers.expert_sum_device(x, 0, positions, weights, x, 0, out, t, 1, width, BF16,
                                    now()) == 1
    assert all_rows(out, 3 * x)


def test_dot_products(torch_cuda):
    """4.3 million tokens, one to a wave."""
    t, width = 4300001, 264
    x = line(width)
    positions = torch.arange(t, dtype=torch.int32, device="cuda")
    positions[-1] = -1
    dx = torch.full((t, width), 7.0, dtype=torch.bfloat16, device="cuda")
    dweights = torch.full((t, 1), 7.0, device="cuda")
    assert layers.expert_rows_backward_device(x, 0, x, 0, positions, None, dx, dweights, t, 1,
                                              width, BF16, now()) == 1
    assert all_rows(dx[:-1], x) and (dx[-1] == 0).all()
    # Sums of whole numbers below 2^24: exact.
    assert (dweights[:-1] == x.float().square().sum()).all() and dweights[-1] == 0


def test_lookup(torch_cuda):
    t, width = 70001, 32000
    table = torch.stack([line(width), -line(width)])
    ids = torch.zeros(t, dtype=torch.int32, device="cuda")
    ids[-1] = 1
    out = torch.full((t, width), 7.0, dtype=torch.bfloat16, device="cuda")
    assert layers.embed_device(ids, table, width * 2, None, 0, 2.0, out, t, 2, width, BF16,
                               now()) == 1
    assert all_rows(out[:-1], 2 * table[0]) and (out[-1] == 2 * table[1]).all()


def test_table_gradient(torch_cuda):
    """2^20 entries in five pieces each."""
    t, entries, width = 100, 2 ** 20, 1100
    ids = torch.full((t,), entries - 1, dtype=torch.int32, device="cuda")
    ids[::2] = 0
    order = torch.empty(t, dtype=torch.int32, device="cuda")
    ranges = torch.empty(entries, 2, dtype=torch.int32, device="cuda")
    space = torch.empty(max(layers.embed_order_workspace_bytes(t, entries),
                            layers.embed_backward_workspace_bytes(t, entries, width)),
                        dtype=torch.uint8, device="cuda")
    dout = line(width).float()
    dtable = torch.full((entries, width), 7.0, device="cuda")
    assert layers.embed_order_device(ids, order, ranges, space, t, entries, now()) == 1
    assert layers.embed_backward_device(dout, 0, ids, order, ranges, 1.0, dtable, space, t,
                                        entries, width, F32, now()) == 1
    assert (dtable[0] == 50 * dout).all() and (dtable[-1] == 50 * dout).all()
    assert all_rows(dtable[1:-1], torch.zeros_like(dout))


def test_order_of_many(torch_cuda):
    """20 million tokens: 256 segments of 78,336, which a wave takes in many turns."""
    t, entries = 20000003, 2 ** 20
    g = torch.Generator("cuda").manual_seed(1)
    ids = torch.randint(-5, entries + 5, (t,), device="cuda", generator=g).int()
    ids[::3] = 77
    order = torch.empty(t, dtype=torch.int32, device="cuda")
    ranges = torch.empty(entries, 2, dtype=torch.int32, device="cuda")
    space = torch.empty(layers.embed_order_workspace_bytes(t, entries), dtype=torch.uint8,
                        device="cuda")
    assert layers.embed_order_device(ids, order, ranges, space, t, entries, now()) == 1
    key = torch.where((ids >= 0) & (ids < entries), ids, entries)
    sort = key.sort(stable=True)
    assert torch.equal(order, torch.where(sort.values < entries, sort.indices, -1).int())
    ends = torch.searchsorted(sort.values, torch.arange(entries + 1, dtype=torch.int32,
                                                        device="cuda"))
    want = torch.stack([ends[:-1], ends[1:]], 1)
    want[want[:, 0] == want[:, 1]] = 0
    assert torch.equal(ranges, want.int())


def test_eight_bit_rows(torch_cuda):
    rows, k = 4300001, 16
    x = torch.ones(rows, k, device="cuda")
    x[-1] = -2
    codes = torch.full((rows, 128), 7, dtype=torch.int8, device="cuda")
    scales = torch.empty(rows, device="cuda")
    assert layers.int8_quantise_device(x, k * 4, codes, scales, rows, k, F32, now()) == 1
    assert (codes[:-1, :k] == 127).all() and (codes[:, k:] == 0).all()
    assert (codes[-1, :k] == -127).all()
    assert (scales[:-1] == torch.tensor(1.0) / torch.tensor(127.0)).all()
    assert scales[-1] == torch.tensor(2.0) / torch.tensor(127.0)
    del x, codes, scales
    # The values: 36 million rows of eight pieces.
    rows, k = 36000001, 64
    codes = torch.zeros(rows, 128, dtype=torch.int8, device="cuda")
    codes[-1, :k], codes[rows // 2, :k] = 3, -5
    scales = torch.ones(rows, device="cuda")
    values = torch.full((rows, k), 7.0, dtype=torch.bfloat16, device="cuda")
    assert layers.int8_values_device(codes, scales, values, rows, k, BF16, now()) == 1
    assert (values[-1] == 3).all() and (values[rows // 2] == -5).all()
    assert values.count_nonzero() == 2 * k
