"""Embeddings (hip_layers.h): lookup against 64 bits, the order against a stable
sort, the gradient against sums in 64 bits and against differences; ids that
have no entry, entries without tokens, one entry in every token, odd widths,
strides, graphs, streams.

Tolerances, u = 2^-24.  A looked-up value is one fused product and sum: u of it,
then the type's rounding.  A gradient adds at most 64 rows in turn, the sums of
such runs in at least 16 groups and those after one another, and scales once:
depth 64 + count / 512 + 20.
"""
from __future__ import annotations

import pytest
import torch

from turbinator_c_amd import layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def now():
    return torch.cuda.current_stream()


def spread(g, m, d, dtype, pitch=None, shift=0):
    pitch = pitch or d
    x = torch.full((m * pitch + shift,), float("nan"))
    x[shift:].view(m, pitch)[:, pitch - d:] = torch.randn((m, d), generator=g)
    return x.to(dtype).cuda()[shift:].view(m, pitch)[:, pitch - d:]


def ids_of(g, t, v, kind):
    if kind == "one":
        return torch.full((t,), v // 2, dtype=torch.int32)
    if kind == "none":
        return torch.full((t,), -1, dtype=torch.int32)
    if kind == "rising":
        return (torch.arange(t) * v // t).int()
    ids = torch.randint(0, v, (t,), generator=g)
    if kind == "skewed":
        ids = torch.where(torch.rand(t, generator=g) < 0.4, v - 1, ids)
        ids = torch.where(torch.rand(t, generator=g) < 0.1, 0, ids)
    if kind == "outside":
        far = torch.tensor([-1, -2 ** 31, v, v + 1, 2 ** 31 - 1])
        ids = torch.where(torch.rand(t, generator=g) < 0.3,
                          far[torch.randint(0, 5, (t,), generator=g)], ids)
    return ids.int()


def order_of(ids, entries, stream=None):
    t = len(ids)
    order = torch.full((t + 16,), 77, dtype=torch.int32, device="cuda")
    ranges = torch.full((entries + 8, 2), 77, dtype=torch.int32, device="cuda")
    need = layers.embed_order_workspace_bytes(t, entries)
    space = torch.full((need + 64,), 0xa5, dtype=torch.uint8, device="cuda")
    assert layers.embed_order_device(ids, order, ranges, space, t, entries,
                                     stream or now()) == 1
    torch.cuda.synchronize()
    assert (order[t:] == 77).all() and (ranges[entries:] == 77).all()
    assert (space[need:] == 0xa5).all()
    return order[:t], ranges[:entries]


def plain_order(ids, entries):
    known = (ids >= 0) & (ids < entries)
    key = torch.where(known, ids, entries).long()
    sort = key.sort(stable=True)
    order = torch.where(sort.values < entries, sort.indices, -1)
    ends = torch.searchsorted(sort.values, torch.arange(entries + 1))
    ranges = torch.stack([ends[:-1], ends[1:]], 1)
    return order.int(), torch.where((ranges[:, :1] == ranges[:, 1:]), 0, ranges).int()


def check_order(ids, entries):
    order, ranges = order_of(ids.cuda(), entries)
    want_order, want_ranges = plain_order(ids, entries)
    assert torch.equal(order.cpu(), want_order)
    assert torch.equal(ranges.cpu(), want_ranges)
    return order, ranges


def check_lookup(g, ids, entries, d, dtype, base, pitch, shift):
    t, scale = len(ids), 1.7
    table = spread(g, entries, d, dtype, pitch, shift)
    under = spread(g, t, d, dtype, pitch and pitch + 1, shift) if base else None
    buffer = torch.full((t * d + 64,), 7.0, dtype=dtype, device="cuda")
    assert layers.embed_device(ids.cuda(), table, table.stride(0) * dtype.itemsize, under,
                               under.stride(0) * dtype.itemsize if base else 0, scale, buffer, t,
                               entries, d, layers.DTYPES[dtype], now()) == 1
    known = (ids >= 0) & (ids < entries)
    want = table.cpu().double()[torch.where(known, ids, 0).long()]
    want = torch.where(known[:, None], want * float(torch.tensor(scale)), 0.0)
    if base:
        want = want + under.cpu().double()
    got = buffer[:t * d].view(t, d).cpu().double()
    assert ((got - want).abs() <=
            ((U if dtype != torch.float32 else 0) + HALF[dtype]) * want.abs() * 1.01 +
            LEAST[dtype]).all()
    assert (buffer[-64:] == 7).all()


def backward(ids, order, ranges, dout, scale, entries, stream=None):
    t, d = dout.shape
    need = layers.embed_backward_workspace_bytes(t, entries, d)
    space = torch.full((need + 64,), 0xa5, dtype=torch.uint8, device="cuda")
    buffer = torch.full((entries * d + 64,), 7.0, device="cuda")
    assert layers.embed_backward_device(dout, dout.stride(0) * dout.element_size(), ids, order,
                                        ranges, scale, buffer, space, t, entries, d,
                                        layers.DTYPES[dout.dtype], stream or now()) == 1
    torch.cuda.synchronize()
    assert (buffer[-64:] == 7).all() and (space[need:] == 0xa5).all()
    return buffer[:entries * d].view(entries, d)


def check_backward(g, ids, entries, d, dtype, pitch, shift, order, ranges):
    t, scale = len(ids), 0.6
    dout = spread(g, t, d, dtype, pitch, shift)
    known = (ids >= 0) & (ids < entries)
    # Rows of tokens without an entry are not read.
    dout[~known.cuda()] = float("nan")
    got = backward(ids.cuda(), order, ranges, dout, scale, entries).cpu().double()
    at, rows = ids[known].long(), dout.cpu().double()[known]
    s = float(torch.tensor(scale))
    want = torch.zeros(entries, d, dtype=torch.float64).index_add_(0, at, rows) * s
    size = torch.zeros(entries, d, dtype=torch.float64).index_add_(0, at, rows.abs()) * s
    count = torch.bincount(at, minlength=entries)[:, None]
    bound = (64 + count / 512 + 20) * U * size * 1.001
    assert ((got - want).abs() <= bound).all()


CASES = [(1, 1, 1, "even"), (1, 1000, 5, "even"), (2, 3, 8, "one"), (31, 4, 7, "skewed"),
         (33, 1, 16, "one"), (64, 64, 256, "even"), (65, 5, 33, "outside"), (100, 7, 9, "none"),
         (1000, 300, 130, "skewed"), (1024, 64, 256, "even"), (2048, 2000, 24, "rising"),
         (4096, 1, 12, "one"), (4097, 1024, 20, "skewed"), (5000, 1025, 31, "outside"),
         (6000, 2, 520, "skewed"), (9001, 9001, 17, "even"), (20000, 70000, 8, "skewed"),
         (30011, 3, 40, "one"), (5000, 2 ** 20, 2, "even"), (12000, 40, 65, "rising"),
         (7000, 100, 4, "none")]


@pytest.mark.parametrize("t,entries,d,kind", CASES)
def test_all(torch_cuda, t, entries, d, kind):
    g = torch.Generator().manual_seed(t + entries + d)
    ids = ids_of(g, t, entries, kind)
    order, ranges = check_order(ids, entries)
    for dtype in TYPES:
        check_lookup(g, ids, entries, d, dtype, False, None, 0)
        check_lookup(g, ids, entries, d, dtype, True, d + 3, 1)
        check_backward(g, ids, entries, d, dtype, None, 0, order, ranges)
        check_backward(g, ids, entries, d, dtype, d + 1, 1, order, ranges)


@pytest.mark.parametrize("t,entries", [(70001, 1), (70001, 2), (70001, 1024), (70001, 1025),
                                       (70001, 65536), (600000, 50000), (2 ** 20 + 1, 2 ** 20)])
def test_long_orders(torch_cuda, t, entries):
    for kind in ("even", "skewed", "outside"):
        g = torch.Generator().manual_seed(t)
        check_order(ids_of(g, t, entries, kind), entries)


@pytest.mark.parametrize("kind", ["even", "skewed", "one", "none", "rising", "outside"])
@pytest.mark.parametrize("entries", [1, 127, 128, 4096, 4097, 2 ** 20])
@pytest.mark.parametrize("t", [63, 65, 2047, 2049, 3000, 4095])
def test_short_orders(torch_cuda, t, entries, kind):
    """Around the bounds between ranking, a workgroup's sort and sorting by launches."""
    check_order(ids_of(torch.Generator().manual_seed(t + entries), t, entries, kind), entries)


@pytest.mark.parametrize("count", [31, 32, 33, 63, 64, 65, 95, 96, 97, 128, 129])
def test_ranges_around_a_chunk(torch_cuda, count):
    """Entries whose ranges begin and end at every place of a chunk."""
    g = torch.Generator().manual_seed(count)
    sizes = [count, 1, count + 1, 2, count - 1, 5, count, count, 0, 3, count + 2] * 3
    ids = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes)).int()
    order, ranges = check_order(ids, len(sizes))
    for d in (3, 64, 100, 1030):
        check_backward(g, ids, len(sizes), d, torch.float32, None, 0, order, ranges)
        check_backward(g, ids, len(sizes), d, torch.bfloat16, None, 0, order, ranges)


def test_wide_rows_of_one_entry(torch_cuda):
    g = torch.Generator().manual_seed(1)
    for t, d in ((3000, 2051), (300, 4097)):
        ids = ids_of(g, t, 3, "one")
        order, ranges = check_order(ids, 3)
        check_backward(g, ids, 3, d, torch.bfloat16, None, 0, order, ranges)


def test_broadcast_rows(torch_cuda):
    """Strides of 0: one base row for all tokens, one gradient row for all."""
    g = torch.Generator().manual_seed(2)
    t, entries, d = 300, 20, 50
    ids = ids_of(g, t, entries, "skewed")
    order, ranges = check_order(ids, entries)
    row = spread(g, 1, d, torch.float32)
    table = spread(g, entries, d, torch.float32)
    out = torch.empty(t, d, device="cuda")
    assert layers.embed_device(ids.cuda(), table, d * 4, row, 0, 1.0, out, t, entries, d, 0,
                               now()) == 1
    assert torch.equal(out, table[ids.cuda().long()] + row)
    dtable = torch.empty(entries, d, device="cuda")
    space = torch.empty(layers.embed_backward_workspace_bytes(t, entries, d), dtype=torch.uint8,
                        device="cuda")
    assert layers.embed_backward_device(row, 0, ids.cuda(), order, ranges, 1.0, dtable, space, t,
                                        entries, d, 0, now()) == 1
    count = torch.bincount(ids.long(), minlength=entries).double()[:, None]
    want = count * row.cpu().double()
    assert ((dtable.cpu().double() - want).abs() <= 90 * U * want.abs()).all()


def test_infinities_stay_in_their_entry(torch_cuda):
    g = torch.Generator().manual_seed(3)
    ids = ids_of(g, 500, 6, "even")
    order, ranges = check_order(ids, 6)
    dout = spread(g, 500, 24, torch.float32)
    bad = int((ids == 2).nonzero()[3, 0])
    dout[bad, 1], dout[bad, 2] = float("inf"), float("nan")
    got = backward(ids.cuda(), order, ranges, dout, 1.0, 6)
    assert got[2, 1] == float("inf") and got[2, 2].isnan()
    got[2, 1:3] = 0
    assert got.isfinite().all()


@pytest.mark.parametrize("t", [500, 9000])
def test_ranges_past_the_order_hold_nothing(torch_cuda, t):
    """Ranges that start behind the last place, up to the largest: no tokens."""
    g = torch.Generator().manual_seed(9)
    ids = ids_of(g, t, 40, "even")
    order, ranges = check_order(ids, 40)
    dout = spread(g, t, 40, torch.float32)
    want = backward(ids.cuda(), order, ranges, dout, 1.0, 40)
    most = 2 ** 31 - 1
    ranges[3], ranges[17], ranges[39] = (torch.tensor(r, dtype=torch.int32)
                                         for r in ((most, most), (most - 9, most), (t, most)))
    for entry in (3, 17, 39):
        want[entry] = 0
    assert torch.equal(backward(ids.cuda(), order, ranges, dout, 1.0, 40), want)


def test_gradient_by_differences(torch_cuda):
    """The lookup is linear in the table: central differences are exact but for
    the roundings of the outputs (u of 2 * 4.5 + 4.5 each, times a gradient of
    4.5, in every token of the entry), divided by the step."""
    g = torch.Generator().manual_seed(6)
    t, entries, d, h, scale = 60, 5, 12, 0.25, 2.0
    ids = ids_of(g, t, entries, "skewed")
    order, ranges = check_order(ids, entries)
    table, base, dout = (torch.randn(m, d, generator=g) for m in (entries, t, t))
    grad = backward(ids.cuda(), order, ranges, dout.cuda(), scale, entries).cpu()
    under = base.cuda()

    def value(table):
        out = torch.empty(t, d, device="cuda")
        assert layers.embed_device(ids.cuda(), table.cuda(), d * 4, under, d * 4, scale, out, t,
                                   entries, d, 0, now()) == 1
        return (out.cpu().double() * dout.double()).sum()

    bound = 2 * t * U * 13.5 * 4.5 / (2 * h) + 1e-5
    for i in range(0, entries * d, 5):
        up, down = table.clone(), table.clone()
        up.view(-1)[i] += h
        down.view(-1)[i] -= h
        assert abs(float(value(up) - value(down)) / (2 * h) - float(grad.view(-1)[i])) <= bound


@pytest.mark.parametrize("t", [2000, 9000])
def test_same_every_time_and_on_another_stream(torch_cuda, t):
    g = torch.Generator().manual_seed(7)
    ids = ids_of(g, t, 50, "skewed").cuda()
    dout = spread(g, t, 130, torch.bfloat16)
    order, ranges = order_of(ids, 50)
    first = backward(ids, order, ranges, dout, 1.0, 50)
    side = torch.cuda.Stream()
    side.wait_stream(now())
    for _ in range(3):
        with torch.cuda.stream(side):
            order2, ranges2 = order_of(ids, 50, side)
            again = backward(ids, order2, ranges2, dout, 1.0, 50, side)
        torch.cuda.synchronize()
        assert torch.equal(order, order2) and torch.equal(first, again)


@pytest.mark.parametrize("t", [700, 9000])
def test_graph(torch_cuda, t):
    """The order, lookup and gradient captured once and replayed on other ids,
    one workspace for both, with eager calls between."""
    g = torch.Generator().manual_seed(8)
    entries, d = 1500, 96
    ids = ids_of(g, t, entries, "even").cuda()
    table, dout = spread(g, entries, d, torch.bfloat16), spread(g, t, d, torch.bfloat16)
    out = torch.empty_like(dout)
    order = torch.empty(t, dtype=torch.int32, device="cuda")
    ranges = torch.empty(entries, 2, dtype=torch.int32, device="cuda")
    dtable = torch.empty(entries, d, device="cuda")
    space = torch.empty(max(layers.embed_order_workspace_bytes(t, entries),
                            layers.embed_backward_workspace_bytes(t, entries, d)),
                        dtype=torch.uint8, device="cuda")

    def step():
        s = now()
        assert layers.embed_device(ids, table, d * 2, None, 0, 1.0, out, t, entries, d, 1, s) == 1
        assert layers.embed_order_device(ids, order, ranges, space, t, entries, s) == 1
        assert layers.embed_backward_device(dout, d * 2, ids, order, ranges, 1.0, dtable, space,
                                            t, entries, d, 1, s) == 1

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for kind in ("skewed", "one", "none", "outside"):
        ids.copy_(ids_of(g, t, entries, kind))
        step()
        torch.cuda.synchronize()
        want = out.clone(), order.clone(), ranges.clone(), dtable.clone()
        for b in (out, order, ranges, dtable):
            b.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (out, order, ranges, dtable)))


def test_past_four_gib(torch_cuda):
    """Tables and tokens whose rows lie past 2^32 bytes."""
    t, entries, d = 90000, 300000, 8192
    table = torch.zeros(entries, d, dtype=torch.bfloat16, device="cuda")
    assert table.numel() * 2 > 2 ** 32
    table[-1], table[3] = 2, 1
    ids = torch.full((t,), 3, dtype=torch.int32, device="cuda")
    ids[-5:] = entries - 1
    out = torch.empty(t, d, dtype=torch.bfloat16, device="cuda")
    code = layers.DTYPES[torch.bfloat16]
    assert layers.embed_device(ids, table, d * 2, None, 0, 1.0, out, t, entries, d, code,
                               now()) == 1
    assert (out[:-5] == 1).all() and (out[-5:] == 2).all()
    del table
    t, entries = 300000, 140000
    ids = torch.full((t,), entries - 1, dtype=torch.int32, device="cuda")
    ids[::2] = 1
    dout = torch.ones(t, d, dtype=torch.bfloat16, device="cuda")
    assert dout.numel() * 2 > 2 ** 32 and entries * d * 4 > 2 ** 32
    order, ranges = order_of(ids, entries)
    got = backward(ids, order, ranges, dout, 0.5, entries)
    assert (got[1] == t // 4).all() and (got[-1] == t // 4).all()
    assert (got[0] == 0).all() and (got[2:-1:1000] == 0).all()
